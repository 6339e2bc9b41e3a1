// The last factor of a gated layer (16-bit types): both halves and their product in one tcgen05 kernel.
//
//   h[j, n] = act(sum_k Wg[j, k] Xg[k, n] + bg[j]) * (sum_k Wu[j, k] Xu[k, n] + bu[j])
//
// per block of the pattern, Wg, Wu the two halves of the stacked factor, Xg, Xu the two halves of the
// intermediate (or one shared input).  A tile is 128 x 128 of the output with two fp32 accumulators in tensor
// memory, 128 columns each, double-buffered (all 512 columns): the gate's MMAs, then the up projection's, then
// one commit.  The epilogue reads both accumulators, adds the biases, forms the product in fp32 and rounds
// once, so that neither half goes to memory (training stores both as well, rounded, for the backward pass).
//
// PAIR: two CTAs of a cluster work on one tile of 256 features x 128 batch entries with the two-SM form of the MMA.
// Each holds its own 128 features' weights and accumulators and loads half of the input chunk, so that an SM moves
// half the input from L2 and reads a quarter less shared memory per product (25088 rows of (1,512,192,4): 53 us either
// way, and with both halves kept 93 on single SMs, 75 by pairs; floor 24 from 39.5 GFLOP, 28 from 180 MB; when they are
// used stands at use_pair).  The leading CTA issues the MMAs for both; its
// barriers count both CTAs' copies and epilogue warps.  (Arrivals at the other CTA's barrier carry no cluster-scope
// release: what they order are tensor-memory reads, which have completed; with one, each cost a microsecond.)
//
// Work split, ring, descriptors and epilogue staging are those of tc_kernel.cu: a persistent CTA keeps one tile of
// output features, its weights of both halves resident in shared memory where three k chunks of 64 hold them
// (c <= 192; 96 KB), and walks (block, batch tile) pairs; longer blocks stream weights through the ring.
// The same kernel with one accumulator adds the halves' products instead (kSum): the gradient of a gated layer's
// input, Wg^T dg + Wu^T du, rounded once, in place of two multiplications and an addition.
// Against the halves written by a grouped launch and multiplied by a pass over them, the last factor's traffic
// falls from 2 c + 2 b + 3 b to 2 c + b elements per block and batch entry.
#include <cuda.h>

#include <atomic>

#include "gated.cuh"
#include "gated.h"
#include "tc_epilogue.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace tc {
namespace {

constexpr int kNT = 128, kKC = 64, kBox = 64;    // columns of an accumulator, k per chunk, elements per 128-byte row
constexpr int kChunk = 128 * kKC * 2;            // bytes of one k chunk of either operand
constexpr int kBarBytes = 256;
constexpr int kEpi = 16, kBlock = 64 + kEpi * 32; // epilogue warps, threads

struct Params {
  int a, b, c, d;
  int64_t batch;
  int tiles_n, tiles_j;
  uint32_t rows, row_groups;
  int nk;
  uint32_t idesc;
  const void* bias;
  int dtype, act;
  int stacked_input;  // the halves have an input each
  int* status;
  void* y;            // for outputs stored without a tensor map
  int64_t y_ld;
  int y_direct;       // kRows: batch-last rows that no map can address; kTurned: batch-first, element by element
};

enum { kMapped, kRows, kTurned };
enum { kProduct, kKeep, kSum };  // h; h and both halves; the sum of the halves

template <bool WRES, int NWC, int SX, int STGN, bool PAIR>
struct Cfg {
  static_assert(!PAIR || WRES, "pairs keep their weights");
  static constexpr int kX = kChunk / (PAIR ? 2 : 1);  // a CTA's part of an input chunk
  static constexpr int kStage = 2 * (kX + (WRES ? 0 : kChunk));  // a k chunk of both halves
  static constexpr int kStgPair = STGN * 32 * 128;  // staging of a pair of warps: 32 rows of 128 bytes
  static constexpr int kSmem = 2 * NWC * kChunk + SX * kStage + kEpi / 2 * kStgPair + kBarBytes + 1024;
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(8 * (2 * SX + 6) + 8 <= kBarBytes, "barrier area");
};

// ---- two CTAs of a cluster ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// the address of this CTA's shared variable in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// loads into this CTA's shared memory whose bytes count at a barrier of either CTA
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void pair_load_4d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives at the barrier at this offset in both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t slot_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_smem), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// act(g) * u for two values each, for results that are rounded to 16 bits.  SiLU's factor is 1 / (1 + 2^s), which goes to
// 0 with 2^-s however far below 0 the gate is, and keeps a NaN to itself.  (One reciprocal for two values, 1 / p = q / (p q),
// saves a quarter of the special-function unit's work and takes as many instructions more: 25088 rows 768 -> 2048
// bf16 93.5 us either way.)
template <int ACT>
__device__ __forceinline__ void gate_2(float g0, float g1, float u0, float u1, float& h0, float& h1) {
  if constexpr (ACT == KSMM_ACT_SILU) {
    const uint64_t g = pack_f2(g0, g1);
    float s0, s1, p0, p1;
    unpack_f2(mul_f2(g, pack_f2(-1.4426950409f, -1.4426950409f)), s0, s1);
    unpack_f2(add_f2(pack_f2(exp2_ftz(s0), exp2_ftz(s1)), pack_f2(1.f, 1.f)), p0, p1);
    unpack_f2(mul_f2(mul_f2(pack_f2(rcp_ftz(p0), rcp_ftz(p1)), g), pack_f2(u0, u1)), h0, h1);
  } else if constexpr (ACT == KSMM_ACT_GELU) {
    uint32_t r0 = __float_as_uint(g0), r1 = __float_as_uint(g1);
    gelu_16bit_2(r0, r1);
    h0 = __uint_as_float(r0) * u0;
    h1 = __uint_as_float(r1) * u1;
  } else {
    h0 = gate_value<true>(g0, ACT) * u0;
    h1 = gate_value<true>(g1, ACT) * u1;
  }
}

template <int ACT>
__device__ __forceinline__ void gate_16(const uint32_t (&g)[16], const uint32_t (&u)[16], int dtype, uint32_t (&w)[8]) {
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    float h0, h1;
    gate_2<ACT>(__uint_as_float(g[e]), __uint_as_float(g[e + 1]), __uint_as_float(u[e]), __uint_as_float(u[e + 1]), h0, h1);
    w[e / 2] = pack2(h0, h1, dtype);
  }
}

// r[e] += b for 16 values of a row
__device__ __forceinline__ void add_row_bias(uint32_t (&r)[16], float b) {
  const uint64_t b2 = pack_f2(b, b);
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    float y0, y1;
    unpack_f2(add_f2(pack_f2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), b2), y0, y1);
    r[e] = __float_as_uint(y0);
    r[e + 1] = __float_as_uint(y1);
  }
}

// r[e] += bias[at + e] for 16 columns of a batch-first tile, of which `exist` exist (a multiple of 8): every lane
// reads the same 16 bytes, one transaction per eight columns
__device__ __forceinline__ void add_column_bias(uint32_t (&r)[16], const void* bias, int64_t at, int exist, int dtype) {
  const uint16_t* bp = static_cast<const uint16_t*>(bias) + at;
  const bool whole = (reinterpret_cast<uintptr_t>(bp) & 15) == 0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (c * 8 >= exist) break;
    uint32_t w[4];
    if (whole) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(bp + c * 8));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = static_cast<uint32_t>(__ldg(bp + c * 8 + 2 * e)) | (static_cast<uint32_t>(__ldg(bp + c * 8 + 2 * e + 1)) << 16);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float b0, b1;
      if (dtype == KSMM_BF16) {
        b0 = __uint_as_float(w[e] << 16);
        b1 = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        b0 = __half2float(__ushort_as_half(static_cast<uint16_t>(w[e] & 0xffffu)));
        b1 = __half2float(__ushort_as_half(static_cast<uint16_t>(w[e] >> 16)));
      }
      uint32_t& r0 = r[c * 8 + 2 * e];
      uint32_t& r1 = r[c * 8 + 2 * e + 1];
      r0 = __float_as_uint(__uint_as_float(r0) + b0);
      r1 = __float_as_uint(__uint_as_float(r1) + b1);
    }
  }
}

// IN_LAST / OUT_LAST: layouts of input and output as in tc_kernel.cu.
template <bool IN_LAST, bool OUT_LAST, bool WRES, int NWC, int SX, int STGN, int MODE, bool PAIR>
__global__ void __launch_bounds__(kBlock, 1)
    gated_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmH, const Params P) {
  static_assert(!PAIR || OUT_LAST, "pairs split the features, rows of the accumulator");
  using C = Cfg<WRES, NWC, SX, STGN, PAIR>;
  constexpr bool KEEP = MODE == kKeep, SUM = MODE == kSum;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t wres0 = (raw + 1023u) & ~1023u;  // 1024-byte alignment for the 128-byte swizzle
  const uint32_t ring0 = wres0 + 2 * NWC * kChunk;
  const uint32_t stg0 = ring0 + SX * C::kStage;
  const uint32_t bar0 = stg0 + kEpi / 2 * C::kStgPair;
  uint8_t* bar_gen = smem_raw + (bar0 - raw);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (SX + s); };
  const uint32_t wfull_bar = bar0 + 8u * (2 * SX), wempty_bar = wfull_bar + 8u;
  auto tfull_bar = [&](int q) { return bar0 + 8u * (2 * SX + 2 + q); };
  auto tempty_bar = [&](int q) { return bar0 + 8u * (2 * SX + 4 + q); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bar_gen + 8 * (2 * SX + 6));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 8 * (2 * SX + 6) + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SX; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(wfull_bar, 1);
    mbar_init(wempty_bar, 1);
    for (int q = 0; q < 2; ++q) {
      mbar_init(tfull_bar(q), 1);
      mbar_init(tempty_bar(q), PAIR ? 2 * kEpi : kEpi);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmX);
    prefetch_tensormap(&tmW);
    prefetch_tensormap(&tmY);
    if (KEEP) prefetch_tensormap(&tmH);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      pair_tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    } else {
      tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // (the other CTA's barriers are set up)
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  // barriers that count for both CTAs are the leader's
  auto lead = [&](uint32_t bar) { return PAIR ? map_rank(bar, 0) : bar; };
  (void)lead;
  grid_dep_wait();
  grid_dep_launch();

  const uint32_t d = P.d;
  const int nk = P.nk;
  // (PAIR: tiles_j counts pairs of feature tiles)
  const uint32_t unit = PAIR ? blockIdx.x / 2 : blockIdx.x;
  const int tj = PAIR ? static_cast<int>(unit % P.tiles_j * 2 + rank) : static_cast<int>(unit % P.tiles_j);
  const uint32_t rc = unit / P.tiles_j;
  const uint32_t row_begin = static_cast<uint32_t>(static_cast<uint64_t>(rc) * P.rows / P.row_groups);
  const uint32_t row_end = static_cast<uint32_t>(static_cast<uint64_t>(rc + 1) * P.rows / P.row_groups);
  const int j0 = tj * 128;
  const int blocks = P.a * P.d;

  if (warp == 0) {
    // ===================== TMA producer =====================
    // (the whole warp walks the loop and one elected lane issues, as below)
    const bool one = elect_one();
    uint32_t si = 0, sph = 0, wph = 0;
    int cur_blk = -1;
    bool ok = true;
    auto load_w = [&](uint32_t dst, uint32_t bar, int kc, int blk) {
#pragma unroll
      for (int wb = 0; wb < 2; ++wb) {
        if constexpr (PAIR) pair_load_3d(dst + wb * kKC * 128, &tmW, bar, j0 + wb * kBox, kc * kKC, blk);
        else tma_load_3d(dst + wb * kKC * 128, &tmW, bar, j0 + wb * kBox, kc * kKC, blk);
      }
    };
    // one input of a shared pair is loaded once and read by both halves' MMAs
    const int inputs = P.stacked_input ? 2 : 1;
    const uint32_t stage_bytes = (PAIR ? 2 : 1) * (inputs * C::kX + (WRES ? 0 : 2 * kChunk));
    const uint32_t wfull_lead = lead(wfull_bar);
    for (uint32_t row = row_begin; row < row_end && ok; ++row) {
      const int blk = static_cast<int>(row / P.tiles_n);
      const int n0 = static_cast<int>(row % P.tiles_n) * 128 + (PAIR ? static_cast<int>(rank) * 64 : 0);
      const int i = blk / d, l = blk % d;
      if (WRES && blk != cur_blk) {
        ok = __all_sync(0xffffffffu, mbar_wait<64>(wempty_bar, wph ^ 1u, abort_flag, P.status, kGatedWaits + 0));
        if (!ok) break;
        wph ^= 1u;
        if (one) {
          if (rank == 0) mbar_expect_tx(wfull_bar, (PAIR ? 4 : 2) * nk * kChunk);
          for (int g = 0; g < 2; ++g)
            for (int kc = 0; kc < nk; ++kc) load_w(wres0 + (g * NWC + kc) * kChunk, wfull_lead, kc, blk + g * blocks);
        }
        cur_blk = blk;
      }
      for (int kc = 0; kc < nk; ++kc) {
        ok = __all_sync(0xffffffffu, mbar_wait<64>(empty_bar(si), sph ^ 1u, abort_flag, P.status, kGatedWaits + 1));
        if (!ok) break;
        const uint32_t dst = ring0 + si * C::kStage, bar = lead(full_bar(si));
        if (one) {
          if (rank == 0) mbar_expect_tx(full_bar(si), stage_bytes);
          for (int g = 0; g < inputs; ++g) {
            const uint32_t at = dst + g * C::kX;
            if constexpr (PAIR) {
              // this CTA's 64 of the tile's 128 batch entries
              if constexpr (IN_LAST) pair_load_4d(at, &tmX, bar, n0, l, kc * kKC, i + g * P.a);
              else pair_load_3d(at, &tmX, bar, kc * kKC, i, n0 + g * static_cast<int>(P.batch));
            } else if constexpr (IN_LAST) {
#pragma unroll
              for (int xb = 0; xb < 2; ++xb)
                tma_load_4d(at + xb * kKC * 128, &tmX, bar, n0 + xb * kBox, l, kc * kKC, i + g * P.a);
            } else {
              tma_load_3d(at, &tmX, bar, kc * kKC, i, n0 + g * static_cast<int>(P.batch));
            }
          }
          if (!WRES) {
            for (int g = 0; g < 2; ++g) load_w(dst + 2 * C::kX + g * kChunk, bar, kc, blk + g * blocks);
          }
        }
        if (++si == SX) { si = 0; sph ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    // (The warp walks the loop and one elected lane issues.  25088 rows of (1,512,192,4), batch-last: 70 us with the loop
    // inside `if (lane == 0)`, 59 so, 54 with both halves' chunks in one ring stage.)
    if (rank == 0) {
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t kLboMN = static_cast<uint32_t>((kKC * 128) >> 4) << 16, kLboK = 1u << 16;
      constexpr uint32_t kStepMN = (16 * 128) >> 4, kStepK = (16 * 2) >> 4;
      constexpr unsigned kAll = 0xffffffffu;
      const bool one = elect_one();
      uint32_t si = 0, sph = 0, wph = 0, ut = 0;
      int cur_blk = -1;
      bool ok = true;
      auto commit = [&](uint32_t bar) {
        if (one) {
          if constexpr (PAIR) pair_commit(bar);
          else umma_commit(bar);
        }
      };
      for (uint32_t row = row_begin; row < row_end && ok; ++row, ++ut) {
        const int blk = static_cast<int>(row / P.tiles_n);
        if (WRES && blk != cur_blk) {
          ok = __all_sync(kAll, mbar_wait<0>(wfull_bar, wph, abort_flag, P.status, kGatedWaits + 2));
          if (!ok) break;
          wph ^= 1u;
          cur_blk = blk;
        }
        const uint32_t buf = ut & 1u, bph = (ut >> 1) & 1u;
        ok = __all_sync(kAll, mbar_wait<0>(tempty_bar(buf), bph ^ 1u, abort_flag, P.status, kGatedWaits + 3));
        if (!ok) break;
        tc_fence_after();
        const uint32_t half_x = P.stacked_input ? C::kX : 0;
        for (int kc = 0; kc < nk; ++kc) {
          ok = __all_sync(kAll, mbar_wait<0>(full_bar(si), sph, abort_flag, P.status, kGatedWaits + 4));
          if (!ok) break;
          const uint32_t stage = ring0 + si * C::kStage;
          if (one) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const uint32_t dcol = tmem_base + buf * 2 * kNT + (SUM ? 0 : g * kNT);
              const uint32_t xsrc = stage + g * half_x;
              const uint32_t wsrc = WRES ? wres0 + (g * NWC + kc) * kChunk : stage + 2 * C::kX + g * kChunk;
              const uint32_t xlo = (xsrc >> 4) | (IN_LAST ? kLboMN : kLboK), wlo = (wsrc >> 4) | kLboMN;
#pragma unroll
              for (int k = 0; k < kKC / 16; ++k) {
                const uint64_t xdesc = (static_cast<uint64_t>(kDescHi) << 32) | (xlo + k * (IN_LAST ? kStepMN : kStepK));
                const uint64_t wdesc = (static_cast<uint64_t>(kDescHi) << 32) | (wlo + k * kStepMN);
                const uint32_t more = k != 0 || kc != 0 || (SUM && g != 0) ? 1u : 0u;
                if constexpr (PAIR) pair_umma(dcol, wdesc, xdesc, P.idesc, more);
                else umma<2>(dcol, OUT_LAST ? wdesc : xdesc, OUT_LAST ? xdesc : wdesc, P.idesc, more);
              }
            }
          }
          commit(empty_bar(si));
          if (++si == SX) { si = 0; sph ^= 1u; }
        }
        if (!ok) break;
        commit(tfull_bar(buf));
        if (WRES && (row + 1 == row_end || static_cast<int>((row + 1) / P.tiles_n) != blk)) commit(wempty_bar);
      }
    }
    __syncwarp();
  } else {
    // ===================== epilogue =====================
    // Sixteen warps, four per scheduler, with 16 columns of both halves in registers at a time.  Warp w: TMEM lane quarter w mod 4, 32 columns
    // of both halves; two warps fill one staging tile of 64 columns, and the first of them stores it.
    const int ew = warp - 2, q = warp & 3, box = ew >> 2;
    const int pair = q + 4 * (box >> 1), side = box & 1;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t stg_base = stg0 + pair * C::kStgPair;
    const int64_t bias_half = static_cast<int64_t>(blocks) * P.b;
    uint32_t ut = 0, sti = 0;
    int bias_blk = -1;
    float bg = 0.f, bu = 0.f;  // batch-last: the biases of this lane's row, loaded when the block changes
    for (uint32_t row = row_begin; row < row_end; ++row, ++ut) {
      const int blk = static_cast<int>(row / P.tiles_n);
      const int n0 = static_cast<int>(row % P.tiles_n) * 128;
      const int i = blk / d, l = blk % d;
      const uint32_t buf = ut & 1u, bph = (ut >> 1) & 1u;
      const int row_limit = OUT_LAST ? P.b - j0 : static_cast<int>(min(P.batch - n0, static_cast<int64_t>(128)));
      const int col_limit = OUT_LAST ? static_cast<int>(min(P.batch - n0, static_cast<int64_t>(kNT))) : P.b - j0;
      if (OUT_LAST && !SUM && P.bias != nullptr && blk != bias_blk) {
        if (q * 32 + lane < row_limit) {
          const int64_t at = (static_cast<int64_t>(i) * P.b + j0 + q * 32 + lane) * d + l;
          bg = bias_at(P.bias, at, P.dtype);
          bu = bias_at(P.bias, at + bias_half, P.dtype);
        }
        bias_blk = blk;
      }
      int got = 1;
      if (lane == 0) got = mbar_wait<64>(tfull_bar(buf), bph, abort_flag, P.status, kGatedWaits + 5) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) break;
      tc_fence_after();
      const int col0 = (box >> 1) * 64;     // of the pair's staging tile
      const bool active = q * 32 < row_limit && col0 < col_limit;  // (the same for both warps of a pair)
      const uint32_t t0 = tmem_base + lane_addr + buf * 2 * kNT + box * 32;
      // the accumulators have been read: hand them back
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) arrive_at(lead(tempty_bar(buf)));
          else mbar_arrive(tempty_bar(buf));
        }
      };
      if (!active) {
        release();
        continue;
      }
      // 16 columns from s * 16 on of either half, with its bias
      auto take_g = [&](uint32_t (&r)[16], int s) {
        if (SUM || P.bias == nullptr) return;
        if constexpr (OUT_LAST) add_row_bias(r, bg);
        else add_column_bias(r, P.bias, static_cast<int64_t>(i) * P.b + j0 + box * 32 + s * 16, col_limit - box * 32 - s * 16, P.dtype);
      };
      auto take_u = [&](uint32_t (&r)[16], int s) {
        if (P.bias == nullptr) return;
        if constexpr (OUT_LAST) add_row_bias(r, bu);
        else add_column_bias(r, P.bias, bias_half + static_cast<int64_t>(i) * P.b + j0 + box * 32 + s * 16,
                             col_limit - box * 32 - s * 16, P.dtype);
      };
      uint32_t stg = 0;
      // the pair's next staging tile, once the store that used it last has read it
      auto next_tile = [&]() {
        stg = stg_base + (STGN > 1 ? sti * 4096u : 0u);
        if (STGN > 1) sti = (sti + 1 == STGN) ? 0u : sti + 1;
        if (side == 0 && lane == 0) bulk_wait_read<STGN - 1>();
        bar_sync_named(1 + pair, 64);
      };
      auto fill = [&](const uint32_t (&w)[8], int s) {
#pragma unroll
        for (int ch = 0; ch < 2; ++ch)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stg + lane * 128 + (((side * 4 + s * 2 + ch) ^ (lane & 7)) << 4)),
                       "r"(w[4 * ch]), "r"(w[4 * ch + 1]), "r"(w[4 * ch + 2]), "r"(w[4 * ch + 3])
                       : "memory");
      };
      auto send = [&](const CUtensorMap* tm, int half) {
        fence_proxy_async();
        bar_sync_named(1 + pair, 64);
        if (side == 0 && lane == 0) {
          if constexpr (OUT_LAST) tma_store_4d(tm, stg, n0 + col0, l, j0 + q * 32, i + half * P.a);
          else tma_store_4d(tm, stg, j0 + col0, i, n0 + q * 32, half);
          bulk_commit();
        }
      };
      if constexpr (KEEP) {
        // (Rounded to the layer's type, as every intermediate of a chain is: fp32 halves would be 8 bytes an element in place
        // of 4, written here and read by the backward.  The product is formed from the unrounded halves.)
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          next_tile();
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            uint32_t r[16], w[8];
            tmem_ld16(t0 + half * kNT + s * 16, r);
            tmem_ld_wait();
            if (half) take_u(r, s);
            else take_g(r, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), P.dtype);
            fill(w, s);
          }
          send(&tmH, half);
        }
      }
      const bool turn = OUT_LAST && !SUM && P.y_direct == kTurned;
      if (!turn) next_tile();
      // (rolled up in training, where that costs nothing and saves a fifth of the kernel's code)
      constexpr int kUnroll = KEEP ? 1 : 2;
#pragma unroll kUnroll
      for (int s = 0; s < 2; ++s) {
        uint32_t g[16], w[8];
        tmem_ld16(t0 + s * 16, g);
        if constexpr (SUM) {
          tmem_ld_wait();
          if (s == 1) release();
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]), P.dtype);
        } else {
          uint32_t u[16];
          tmem_ld16(t0 + kNT + s * 16, u);
          tmem_ld_wait();
          if (s == 1) release();
          take_g(g, s);
          take_u(u, s);
          switch (P.act) {
            case KSMM_ACT_SILU: gate_16<KSMM_ACT_SILU>(g, u, P.dtype, w); break;
            case KSMM_ACT_GELU: gate_16<KSMM_ACT_GELU>(g, u, P.dtype, w); break;
            case KSMM_ACT_SIGMOID: gate_16<KSMM_ACT_SIGMOID>(g, u, P.dtype, w); break;
            default: {  // none and relu: a lowest value (a NaN is not below it)
              const float low = P.act == KSMM_ACT_RELU ? 0.f : -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (__uint_as_float(g[e]) < low) g[e] = __float_as_uint(low);
              gate_16<KSMM_ACT_NONE>(g, u, P.dtype, w);
            }
          }
        }
        if (turn) {
          // a lane's 16 batch entries of one feature
          if (q * 32 + lane < row_limit) {
            const int64_t feats = static_cast<int64_t>(blocks) * P.b;
            uint16_t* y = static_cast<uint16_t*>(P.y) + (n0 + box * 32 + s * 16) * feats +
                          (static_cast<int64_t>(i) * P.b + j0 + q * 32 + lane) * d + l;
            const int exist = col_limit - box * 32 - s * 16;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e < exist) y[e * feats] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
          }
        } else {
          fill(w, s);
        }
      }
      if (turn) continue;
      if (OUT_LAST && P.y_direct) {
        // each warp of the pair stores half of the tile's rows
        bar_sync_named(1 + pair, 64);
        uint8_t* yrow = static_cast<uint8_t*>(P.y) +
                        (((static_cast<int64_t>(i) * P.b + j0 + q * 32) * d + l) * P.y_ld + n0 + col0) * 2;
        store_rows<2, 8>(stg, yrow, static_cast<int64_t>(d) * P.y_ld * 2, min(32, row_limit - q * 32), col_limit - col0, lane,
                         16 * side, 16 * side + 16);
        // An empty group for the product's staging tile: next_tile() takes it that every tile handed out has one, and
        // without it would hand out a tile that a half's store is still reading.
        if (KEEP && side == 0 && lane == 0) bulk_commit();
      } else {
        send(&tmY, 0);
      }
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }

  // ===================== teardown =====================
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // neither CTA leaves while the other's MMAs or arrivals reach its shared memory
  if (*abort_flag) {
    // copies that may still be in flight land before the shared memory is handed on
    __nanosleep(20000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) pair_tmem_dealloc(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

template <bool IN_LAST, bool OUT_LAST, bool WRES, int NWC, int SX, int STGN, int MODE, bool PAIR = false>
int launch(const Problem& p, void* halves, int64_t halves_ld, cudaStream_t stream, bool turn = false) {
  using C = Cfg<WRES, NWC, SX, STGN, PAIR>;
  constexpr bool KEEP = MODE == kKeep;
  auto kern = gated_kernel<IN_LAST, OUT_LAST, WRES, NWC, SX, STGN, MODE, PAIR>;
  static std::atomic<bool> attr_set[64];  // once per device (a repeated set is harmless)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess)
      return set_error(KSMM_ERR_CUDA, "cannot reserve %d bytes of shared memory: %s", C::kSmem, cudaGetErrorString(e));
    attr_set[dev] = true;
  }
  const uint64_t a = p.a, b = p.b, c = p.c, d = p.d, B = p.batch, GX = p.group_shared_input ? 1 : 2;
  CUtensorMap tmX, tmW, tmY, tmH;
  int st;
  {
    const uint64_t dims[3] = {b, c, 2 * a * d}, str[3] = {1, b, c * b};
    const uint32_t box[3] = {kBox, kKC, 1};
    if ((st = encode_map(&tmW, p.in_dtype, 3, p.w, dims, str, box)) != KSMM_OK) return st;
  }
  if (IN_LAST) {
    const uint64_t L = in_stride(p), dims[4] = {B, d, c, GX * a}, str[4] = {1, L, d * L, c * d * L};
    const uint32_t box[4] = {kBox, 1, kKC, 1};
    if ((st = encode_map(&tmX, p.in_dtype, 4, p.in, dims, str, box)) != KSMM_OK) return st;
  } else {
    const uint64_t dims[3] = {c, a, GX * B}, str[3] = {1, c, a * c};
    const uint32_t box[3] = {kKC, 1, PAIR ? 64 : 128};
    if ((st = encode_map(&tmX, p.in_dtype, 3, p.in, dims, str, box)) != KSMM_OK) return st;
  }
  Params P = {};
  P.y = p.out;
  P.y_ld = out_stride(p);
  P.y_direct = turn ? kTurned : (OUT_LAST && !rows_addressable(p.out, P.y_ld, 2) ? kRows : kMapped);
  auto output_map = [&](CUtensorMap* tm, const void* ptr, int64_t ld, uint64_t groups) {
    if (OUT_LAST) {
      const uint64_t L = ld, dims[4] = {B, d, b, groups * a}, str[4] = {1, L, d * L, b * d * L};
      const uint32_t box[4] = {kBox, 1, 32, 1};
      return encode_map(tm, p.out_dtype, 4, ptr, dims, str, box);
    }
    const uint64_t dims[4] = {b, a, B, groups}, str[4] = {1, b, a * b, a * b * B};
    const uint32_t box[4] = {kBox, 1, 32, 1};
    return encode_map(tm, p.out_dtype, 4, ptr, dims, str, box);
  };
  tmY = tmH = tmX;  // (unused ones)
  if (!P.y_direct && (st = output_map(&tmY, p.out, P.y_ld, 1)) != KSMM_OK) return st;
  if (KEEP && (st = output_map(&tmH, halves, halves_ld, 2)) != KSMM_OK) return st;
  P.a = p.a; P.b = p.b; P.c = p.c; P.d = p.d;
  P.batch = p.batch;
  P.nk = (p.c + kKC - 1) / kKC;
  P.bias = p.bias;
  P.dtype = p.out_dtype;
  P.act = p.activation;
  P.stacked_input = GX == 2;
  P.status = status_word();
  if (!P.status) return set_error(KSMM_ERR_CUDA, "cannot resolve the device status word");
  const uint32_t fmt = p.in_dtype == KSMM_BF16 ? 1u : 0u;
  const uint32_t a_mn = (OUT_LAST || IN_LAST) ? 1u : 0u, b_mn = (!OUT_LAST || IN_LAST) ? 1u : 0u;
  P.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn << 15) | (b_mn << 16) | (static_cast<uint32_t>(kNT >> 3) << 17) |
            (static_cast<uint32_t>((PAIR ? 256 : 128) >> 4) << 24);
  P.tiles_n = static_cast<int>((B + 127) / 128);
  P.tiles_j = static_cast<int>((b + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
  int sms = num_sms();  // CTAs, or pairs, at the same time
  if constexpr (PAIR) {
    // A pair needs the two SMs of one TPC; ask how many there are rather than run a last pair on its own
    static std::atomic<int> pairs[64];
    int n = dev >= 0 && dev < 64 ? pairs[dev].load(std::memory_order_relaxed) : 0;
    if (!n) {
      cudaLaunchConfig_t q = {};
      q.gridDim = dim3(2);
      q.blockDim = dim3(kBlock);
      q.dynamicSmemBytes = C::kSmem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 2;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      q.attrs = at;
      q.numAttrs = 1;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kern, &q);
      if (e != cudaSuccess || n <= 0)
        return set_error(KSMM_ERR_CUDA, "cannot place pairs of CTAs: %s", cudaGetErrorString(e));
      if (dev >= 0 && dev < 64) pairs[dev].store(n, std::memory_order_relaxed);
    }
    sms = n;
  }
  if (sms <= 0) return set_error(KSMM_ERR_NO_DEVICE, "no CUDA device");
  const int64_t rows = static_cast<int64_t>(P.tiles_n) * p.a * p.d;
  if (rows <= 0 || rows > 0x7fffffffLL || P.tiles_j > sms)
    return set_error(KSMM_ERR_UNSUPPORTED, "gated kernel: %lld rows x %d j tiles exceed the work-split limits",
                     static_cast<long long>(rows), P.tiles_j);
  P.rows = static_cast<uint32_t>(rows);
  const int64_t groups = std::min<int64_t>(sms / P.tiles_j, rows);
  P.row_groups = static_cast<uint32_t>(groups);
  cudaError_t err;
  if constexpr (PAIR) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(groups * P.tiles_j * 2));
    cfg.blockDim = dim3(kBlock);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    err = cudaLaunchKernelEx(&cfg, kern, tmX, tmW, tmY, tmH, P);
  } else {
    err = launch_pdl(kern, static_cast<unsigned>(groups * P.tiles_j), kBlock, C::kSmem, stream, tmX, tmW, tmY, tmH, P);
  }
  count_launch();
  if (err == cudaSuccess) err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "gated kernel launch failed: %s", cudaGetErrorString(err));
  return KSMM_OK;
}

// Two CTAs per tile where that is faster: three chunks of k, features that fill the pairs' tiles, and ten tiles or more
// for every pair of SMs.  Calls of two-factor layers in bf16, 25088 rows if not
// said otherwise, single CTAs against pairs:
//   768 -> 2048, (1,512,192,4) last: 93.1 and 92.5 us, training step 437 and 423; 8192 rows (7 tiles) 34.9 and 35.7
//   768 -> 4096, (1,1024,192,4): 149 and 147, training 710 and 683; 4096 rows (7 tiles) 33.7 and 34.0
//   1536 -> 1600, (1,200,192,8): 122.0 and 121.0, training 495 and 487; 4096 rows 29.0 and 29.6
// and where the rule says single: 512 -> 4096, (1,512,64,8), two chunks less: 110.7 and 112.9; 1024 -> 2816,
// (1,352,128,8), four of six tiles' features exist: 111 and 129; 768 -> 1536, (1,384,192,4), three of four: 78.6 and 89.0.
bool use_pair(const Problem& p) {
  const int64_t tiles = (p.batch + 127) / 128 * p.a * p.d * ((p.b + 255) / 256);
  return p.c > 2 * kKC && p.c <= 3 * kKC && (p.b - 1) % 256 >= 128 && tiles >= 5 * num_sms();
}

template <bool IN_LAST, bool OUT_LAST>
int launch_layout(const Problem& p, void* halves, int64_t halves_ld, cudaStream_t stream, bool turn) {
  if constexpr (OUT_LAST) {
    if (use_pair(p))
      return halves ? launch<IN_LAST, true, true, 3, 4, 2, kKeep, true>(p, halves, halves_ld, stream, turn)
                    : launch<IN_LAST, true, true, 3, 6, 1, kProduct, true>(p, halves, halves_ld, stream, turn);
  }
  if (p.c <= 3 * kKC)
    return halves ? launch<IN_LAST, OUT_LAST, true, 3, 2, 2, kKeep>(p, halves, halves_ld, stream, turn)
                  : launch<IN_LAST, OUT_LAST, true, 3, 3, 1, kProduct>(p, halves, halves_ld, stream, turn);
  if constexpr (IN_LAST && OUT_LAST) {
    return halves ? launch<true, true, false, 0, 2, 2, kKeep>(p, halves, halves_ld, stream, turn)
                  : launch<true, true, false, 0, 2, 1, kProduct>(p, halves, halves_ld, stream, turn);
  }
  return set_error(KSMM_ERR_UNSUPPORTED, "gated kernel: blocks longer than %d keep the batch-last layout", 3 * kKC);
}

template <bool OUT_LAST>
int launch_sum(const Problem& p, cudaStream_t stream) {
  if (p.c <= 3 * kKC) return launch<true, OUT_LAST, true, 3, 3, 1, kSum>(p, nullptr, 0, stream);
  if constexpr (OUT_LAST) return launch<true, true, false, 0, 2, 1, kSum>(p, nullptr, 0, stream);
  return set_error(KSMM_ERR_UNSUPPORTED, "gated kernel: blocks longer than %d keep the batch-last layout", 3 * kKC);
}

}  // namespace
}  // namespace tc

bool tc_gated_fits(const int32_t* q, int64_t batch, int dtype, int in_last, int out_last) {
  if (dtype != KSMM_F16 && dtype != KSMM_BF16) return false;
  // (smaller blocks are bandwidth problems that the register-tiled kernels serve more tightly)
  if (q[1] < 32 || q[2] < 16 || q[1] % 8 != 0 || q[1] > 16384) return false;
  // (longer blocks stream their weights, in one layout only)
  if ((!in_last || !out_last) && (q[3] != 1 || q[2] % 8 != 0 || q[2] > 3 * tc::kKC)) return false;
  return batch > 0 && batch <= 0x3fffffffLL && static_cast<int64_t>(q[0]) * q[3] <= 0x3fffffffLL;
}

int tc_gated_launch(const Problem& p, void* halves, int64_t halves_ld, bool turn, cudaStream_t stream) {
  const bool in_last = in_is_last(p), out_last = out_is_last(p);
  if (in_last) return out_last ? tc::launch_layout<true, true>(p, halves, halves_ld, stream, turn)
                               : tc::launch_layout<true, false>(p, halves, halves_ld, stream, turn);
  return out_last ? tc::launch_layout<false, true>(p, halves, halves_ld, stream, turn)
                  : tc::launch_layout<false, false>(p, halves, halves_ld, stream, turn);
}

int tc_gated_sum(const Problem& p, cudaStream_t stream) {
  return out_is_last(p) ? tc::launch_sum<true>(p, stream) : tc::launch_sum<false>(p, stream);
}

}  // namespace ksmm
