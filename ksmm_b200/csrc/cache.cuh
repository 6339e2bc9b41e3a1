// Attention over a paged cache: what its kernels share (arguments, the split of the work, the partial results).
#pragma once

#include "common.cuh"

namespace ksmm {
namespace cache {

constexpr int kWaits = 110;      // codes of this family's bounded waits: 110 to 119
constexpr int kMaxDim = 256;
constexpr float kNone = -3.402823466e38f;  // a running maximum before the first key: differences of two are 0, not NaN

struct Pool {
  char* data[2];        // keys, values
  float* scales[2];     // 8-bit caches
  int64_t page[2], head[2], token[2];     // strides in elements
  int64_t spage[2], shead[2], stoken[2];  // of the scales
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  int64_t pages, table_stride;
  int page_size, table_width, kv_heads, dim;
  int sequences, tokens, each;  // each: new tokens of a sequence where there are no starts
};

// two e4m3 (the low 16 bits) as fp16
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
  return r;
}

// A sequence as the kernels see it.
struct Sequence {
  int start, n;  // its rows
  int length;    // its tokens, as far as the table has pages for them
  bool bad;      // it is longer than that
};

__device__ __forceinline__ Sequence sequence(const Pool& p, int s) {
  Sequence q;
  if (p.starts) {
    q.start = min(max(p.starts[s], 0), p.tokens);
    q.n = min(max(p.starts[s + 1], q.start), p.tokens) - q.start;
  } else {
    q.start = s * p.each;
    q.n = p.each;
  }
  const int64_t most = static_cast<int64_t>(p.table_width) * p.page_size;
  const int length = max(p.lengths[s], 0);
  q.bad = length > most;
  q.length = q.bad ? static_cast<int>(most) : length;
  return q;
}

struct Attend {
  Pool pool;
  const char* q;
  char* out;
  int64_t q_token, q_head, out_token, out_head;
  int64_t window;       // 0: none
  int heads, group;
  float scale;          // of the scores, times log2(e)
  int clear_rest;
  int tile_rows;        // rows (token, head of the group) of an item
  int unit_log2;        // of the tokens of a unit, the piece in which a cache's length is split
  int least, most;      // sequences with fewer or more rows in a group are another kernel's
  int split;            // an item's units may be several CTAs'
  float* partial;       // split: 2 slots per CTA of tile_rows * (dim + 2) floats
  int64_t* slots;       // split: the item of each slot, or -1
  int* status;
};

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

// An item: up to tile_rows rows of one sequence and one key head.  They are numbered sequence by sequence, then head by head.
struct Work {
  int units, tiles;  // units of an item (of a split launch), items of a head
  int64_t items;     // of the sequence
};

__device__ __forceinline__ int first_key(const Attend& a, const Sequence& q, int row_token) {
  if (!a.window) return 0;
  const int64_t lo = static_cast<int64_t>(q.length) - q.n + row_token - a.window + 1;
  return static_cast<int>(lo < 0 ? 0 : lo);
}

// units up to a token; a length is at most 2^31 - 65537
__device__ __forceinline__ int units_to(const Attend& a, int length) { return (length + (1 << a.unit_log2) - 1) >> a.unit_log2; }

// (Out of line, once: inlined in a dozen places it was three quarters of a kernel's code, and a block's start waited for that to be
// fetched.  In 32 bits where they suffice: 64 take several hundred cycles.)
static __device__ __noinline__ int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// (the host has seen to it that rows and their tiles fit 32 bits)
__device__ __forceinline__ Work work_of(const Attend& a, const Sequence& q) {
  Work w;
  const int rows = q.n * a.group;
  const bool mine = rows >= a.least && rows <= a.most;
  w.tiles = mine ? static_cast<unsigned>(rows + a.tile_rows - 1) / static_cast<unsigned>(a.tile_rows) : 0;
  // (a sequence without keys is a unit of work as well: its rows are zeros)
  w.units = mine ? max(1, units_to(a, q.length) - (first_key(a, q, 0) >> a.unit_log2)) : 0;
  w.items = static_cast<int64_t>(w.tiles) * a.pool.kv_heads;
  return w;
}

// A piece of an item, from a block's share.
struct Segment {
  int64_t item;        // its number, for the partial results
  int s, head, tile;   // s < 0: no more segments
  int start, n;        // the sequence's rows
  int length;          // its tokens
  int bad;             // it is longer than its table
  int lo, hi;          // the keys that the item's rows see lie in [lo, hi)
  int first_position;  // of its first row
  int from, to;        // the units to be gone through, counted from the sequence's first token
  int slot;            // where the result goes: 0 the output, 1 or 2 the block's first or second slot
};

constexpr int kWholeUnits = 8;  // items of up to so many units stay whole where there is a block for each: joining parts costs more

// A block's share, walked segment by segment by ONE warp, all lanes alike: as many units of the launch's, counted sequence by sequence
// and head by head, as every other block's; in a launch without a split, or of few short sequences, one whole item.  The warp hands the
// segments on: what a segment is takes a chain of reads and divisions (several microseconds where every thread followed it).
struct Walker {
  Sequence seq;
  Work work;
  int s, head, tile, from;
  int64_t left;  // units, or whole items
  bool whole;

  __device__ void set(const Attend& a, int which) {
    s = which;
    seq = sequence(a.pool, s);
    work = work_of(a, seq);
  }

  // A lane sums a run of sequences, the warp forms the runs' prefix sums, and the run that holds the block's first unit is walked by
  // its lane.  false: nothing to do (a split block then has marked its slots).
  __device__ bool start(const Attend& a) {
    if (!a.split && !a.pool.starts) {
      // (all sequences have the same number of items)
      const int rows = a.pool.each * a.group;
      const int per = rows < a.least || rows > a.most ? 0 : (rows + a.tile_rows - 1) / a.tile_rows * a.pool.kv_heads;
      const int which = per ? blockIdx.x / static_cast<unsigned>(per) : a.pool.sequences;
      if (which >= a.pool.sequences) return false;
      left = 1;
      whole = true;
      from = 0;
      set(a, which);
      const int item = blockIdx.x - which * per, t = item / a.pool.kv_heads;
      head = item - t * a.pool.kv_heads;
      tile = work.tiles - 1 - t;
      return true;
    }
    constexpr uint32_t kAll = 0xffffffffu;
    const int lane = threadIdx.x % 32;
    const int run = (a.pool.sequences + 31) / 32;
    const int first = min(lane * run, a.pool.sequences), end = min(first + run, a.pool.sequences);
    int64_t units = 0, items = 0;
    int most = 0;
#pragma unroll 1
    for (int i = first; i < end; ++i) {
      const Work w = work_of(a, sequence(a.pool, i));
      units += w.items * w.units;
      items += w.items;
      most = max(most, w.units);
    }
    int64_t units_before = units, items_before = items;
#pragma unroll 1
    for (int d = 1; d < 32; d *= 2) {
      const int64_t u = __shfl_up_sync(kAll, units_before, d), n = __shfl_up_sync(kAll, items_before, d);
      if (lane >= d) {
        units_before += u;
        items_before += n;
      }
    }
    most = __reduce_max_sync(kAll, most);
    const int64_t all_units = __shfl_sync(kAll, units_before, 31), all_items = __shfl_sync(kAll, items_before, 31);
    const int64_t block = blockIdx.x, blocks = gridDim.x;
    whole = !a.split || (most <= kWholeUnits && all_items <= blocks);
    int64_t place = block, last = block + 1, mine = items, before = items_before - items;
    if (!whole) {
      // (with fewer units than blocks the first all_units blocks have one each)
      mine = units;
      before = units_before - units;
      const int64_t n = min(all_units, blocks);
      place = block < n ? divide(block * all_units, n) : all_units;
      last = block < n ? divide((block + 1) * all_units, n) : all_units;
    }
    const uint32_t holds = __ballot_sync(kAll, place < last && place >= before && place < before + mine);
    left = last - place;
    if (!holds) {
      if (a.split && lane < 2) a.slots[2 * block + lane] = -1;
      return false;
    }
    int which = 0;
    int64_t offset = 0;
    if (holds >> lane & 1) {
      for (int i = first; i < end; ++i) {
        const Work w = work_of(a, sequence(a.pool, i));
        const int64_t n = whole ? w.items : w.items * w.units;
        if (place < before + n) {
          which = i;
          offset = place - before;
          break;
        }
        before += n;
      }
    }
    const int holder = __ffs(holds) - 1;
    which = __shfl_sync(kAll, which, holder);
    offset = __shfl_sync(kAll, offset, holder);
    set(a, which);
    const int64_t item = whole ? offset : divide(offset, work.units);
    from = whole ? 0 : static_cast<int>(offset - item * work.units);
    if (a.split) {
      head = static_cast<int>(divide(item, work.tiles));
      tile = static_cast<int>(item - static_cast<int64_t>(head) * work.tiles);
    } else {
      // the last tiles of all heads come first: they see the most keys
      const int64_t t = divide(item, a.pool.kv_heads);
      head = static_cast<int>(item - t * a.pool.kv_heads);
      tile = work.tiles - 1 - static_cast<int>(t);
    }
    return true;
  }

  // the next segment; one with s < 0 where there is none
  __device__ void next(const Attend& a, Segment* g) {
    g->s = -1;
    if (left <= 0) return;
    while (work.items == 0 || head >= a.pool.kv_heads) {
      if (s + 1 >= a.pool.sequences) return;  // (not reached: the units end with the last sequence's)
      set(a, s + 1);
      head = tile = from = 0;
    }
    const int to = whole ? work.units : static_cast<int>(left < work.units - from ? from + left : work.units);
    left -= whole ? 1 : to - from;
    g->item = (static_cast<int64_t>(s) * a.pool.kv_heads + head) << 32 | tile;
    g->s = s;
    g->head = head;
    g->tile = tile;
    g->start = seq.start;
    g->n = seq.n;
    g->length = seq.length;
    g->bad = seq.bad;
    const int t0 = tile * a.tile_rows / a.group;
    g->first_position = seq.length - seq.n + t0;
    g->lo = first_key(a, seq, a.split ? 0 : t0);
    g->hi = seq.length;
    g->from = g->lo >> a.unit_log2;
    if (a.split) {
      // (all tiles of a sequence go through the same units, so that they count the same)
      g->to = g->from + to;
      g->from += from;
    } else {
      const int t1 = ((tile + 1) * a.tile_rows - 1) / a.group;
      g->hi = max(seq.length - seq.n + (t1 < seq.n ? t1 + 1 : seq.n), 0);
      g->to = units_to(a, g->hi);
    }
    // a block's first segment may continue an item, its last may be continued; one that is both is the first
    g->slot = from == 0 && to == work.units ? 0 : from > 0 ? 1 : 2;
    from = to == work.units ? 0 : to;
    if (from == 0 && ++tile == work.tiles) {
      tile = 0;
      ++head;
    }
  }
};

// Reads a word of every 64 bytes of a kernel's parameters, before the wait for the kernel before it: the first use of each such piece
// otherwise waits for it alone, one after the other, in the chain that starts a block.
template <typename P>
__device__ __forceinline__ void touch_parameters(const P& parameters) {
  const int* words = reinterpret_cast<const int*>(&parameters);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(P) / 4); i += 16) asm volatile("" ::"r"(words[i]));
}

// Rows of no sequence, as asked for.
template <typename T>
__device__ void clear_rest(const Attend& a) {
  if (!a.clear_rest || !a.pool.starts) return;
  const int begin = min(max(a.pool.starts[0], 0), a.pool.tokens);
  const int end = min(max(a.pool.starts[a.pool.sequences], begin), a.pool.tokens);
  const int rest = begin + a.pool.tokens - end;
  for (int r = blockIdx.x; r < rest; r += gridDim.x) {
    const int t = r < begin ? r : end + r - begin;
    for (int i = threadIdx.x; i < a.heads * a.pool.dim; i += blockDim.x) {
      const int h = i / a.pool.dim;
      reinterpret_cast<T*>(a.out)[t * a.out_token + h * a.out_head + i - h * a.pool.dim] = ElemTraits<T>::from_float(0.f);
    }
  }
}

// ---------------------------------------------------------------------------
// host side: what the entry points plan with, and the launches (each returns a status)
// ---------------------------------------------------------------------------
constexpr int kMaxBlocks = 512;   // of a split launch (the join kernel's table of weights)

struct TokenShape {
  int blocks, unit;  // blocks on an SM, tokens of a unit
};

// The 16- and 8-bit kernel for few rows.  A step of a warp is a chain (load, products, maximum, exponentials, products) of 1000 to
// 1500 cycles however many tokens it has, and an SM has to pass 23 bytes a cycle: small rows take 32 tokens of a step, wide ones 16.
constexpr int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
constexpr TokenShape token_shape(bool eight, int dp) { return {dp == 256 ? 1 : 2, 4 * (dp == 256 || (!eight && dp == 128) ? 16 : 32)}; }
// Rows of an item.  Sixteen are built for 16-bit caches of up to 128 columns; others go through their keys, the second time in the cache
// of the GPU, once for every eight (each variant is 90 KB of code).
inline int token_rows(int64_t rows, bool eight, int dim) { return rows <= 8 || eight || dim > 128 ? 8 : 16; }

// The fp32 kernel for few rows: rows and tokens of an item's pieces, blocks on an SM.
constexpr int kRowsUnit = 64;
constexpr int kFewRowsTile = 2;
inline int rows_tile(int dim, int64_t rows) { return rows <= kFewRowsTile || dim > 128 ? kFewRowsTile : dim <= 64 ? 8 : 4; }
constexpr int row_blocks(int dim, int tile) { return tile == kFewRowsTile && dim <= 64 ? 2 : 1; }

constexpr int kPlainRows = 8;     // rows of an item in the kernel for what no other takes
constexpr int kFloatRows = 64;    // rows and keys of a tile in the fp32 prompt kernel
inline int prompt_rows(int group) { return 128 / group * group; }

int launch_append(Append& a, int dtype, int cache_dtype, cudaStream_t stream);
int launch_token(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream);
int launch_prompt(const Attend& a, int dtype, bool eight, unsigned grid, cudaStream_t stream);
int launch_float(const Attend& a, unsigned grid, cudaStream_t stream);
int launch_rows(const Attend& a, unsigned grid, cudaStream_t stream);
int launch_plain(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream);
int launch_join(const Attend& a, int dtype, unsigned blocks, int rows, cudaStream_t stream);  // rows: of an item, at most

}  // namespace cache
}  // namespace ksmm
