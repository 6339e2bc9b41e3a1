// Attention over a paged cache: what its kernels share (arguments, the split of the work, the partial results).
#pragma once

#include "common.cuh"

namespace ksmm {
namespace cache {

constexpr int kWaits = 110;      // codes of this family's bounded waits: 110 to 119
constexpr int kUnit = 64;        // tokens of a unit, the piece in which a cache's length is split
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
  int least, most;      // sequences with fewer or more rows in a group are another kernel's
  int split;            // an item's units may be several CTAs'
  float* partial;       // split: 2 slots per CTA of tile_rows * (dim + 2) floats
  int64_t* slots;       // split: the item of each slot, or -1
  int* status;
};

// An item: up to tile_rows rows of one sequence and one key head.  They are numbered sequence by sequence, then head by head; in a
// split launch each counts as its units of kUnit tokens.
struct Work {
  int units, tiles;  // of an item; items of a head
  int64_t weight;    // of the sequence
};

__device__ __forceinline__ int first_key(const Attend& a, const Sequence& q, int row_token) {
  if (!a.window) return 0;
  const int64_t lo = static_cast<int64_t>(q.length) - q.n + row_token - a.window + 1;
  return static_cast<int>(lo < 0 ? 0 : lo);
}

__device__ __forceinline__ Work work_of(const Attend& a, const Sequence& q) {
  Work w;
  const int64_t rows = static_cast<int64_t>(q.n) * a.group;
  if (rows < a.least || rows > a.most) {
    w.units = w.tiles = 0;
    w.weight = 0;
    return w;
  }
  w.tiles = static_cast<int>((rows + a.tile_rows - 1) / a.tile_rows);
  // (a sequence without keys is a unit of work as well: its rows are zeros)
  w.units = a.split ? max(1, (q.length + kUnit - 1) / kUnit - first_key(a, q, 0) / kUnit) : 1;
  w.weight = static_cast<int64_t>(w.units) * w.tiles * a.pool.kv_heads;
  return w;
}

// Finds the sequence that holds place `at(total)` of all sequences' weights.  Every thread of the block calls it; `shared` holds
// 32 + 3 values.  Returns the total; *s and *offset are set to the sequence and the place in it (s = sequences if at >= total).
// A thread sums a run of sequences, the block forms the runs' prefix sums, the run that holds the place is walked by its
// thread: lengths and starts are read once, side by side.
template <int THREADS, typename At>
__device__ int64_t find_place(const Attend& a, int64_t* shared, At at, int* s, int64_t* offset) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int run = (a.pool.sequences + THREADS - 1) / THREADS;
  const int from = min(tid * run, a.pool.sequences), to = min(from + run, a.pool.sequences);
  int64_t sum = 0;
  for (int i = from; i < to; ++i) sum += work_of(a, sequence(a.pool, i)).weight;
  int64_t before = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += v;
  }
  if (lane == 31) shared[warp] = before;
  if (tid == 0) shared[33] = a.pool.sequences;
  __syncthreads();
  constexpr int kWarps = THREADS / 32;
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += shared[w];
    total += shared[w];
  }
  const int64_t place = at(total);
  before -= sum;
  if (sum > 0 && place >= before && place < before + sum) {
    for (int i = from; i < to; ++i) {
      const int64_t w = work_of(a, sequence(a.pool, i)).weight;
      if (place < before + w) {
        shared[33] = i;
        shared[34] = place - before;
        break;
      }
      before += w;
    }
  }
  __syncthreads();
  *s = static_cast<int>(shared[33]);
  *offset = shared[34];
  __syncthreads();  // (the caller may use the array again)
  return total;
}

// A block's share of a split launch, places [begin, end), as segments of items; without a split one item.
struct Segment {
  Sequence seq;
  int s, head, tile;
  int lo, hi;          // the keys that its rows see lie in [lo, hi)
  int first_position;  // of its first row
  int from, to;        // the units to be gone through, counted from the sequence's first token
  int slot;            // where the result goes: 0 the output, 1 or 2 the block's first or second slot
  int64_t item;        // its number, for the partial results
};

struct Share {
  int64_t begin, end, done;
  int s;
  int64_t offset;
  Work work;
  Sequence seq;

  // the next segment, by one thread or by all alike; false where there is none
  __device__ bool next(const Attend& a, Segment* g) {
    if (done >= end) return false;
    while (offset >= work.weight) {
      offset -= work.weight;
      if (++s >= a.pool.sequences) return false;  // (not reached: the places end with the last sequence's)
      seq = sequence(a.pool, s);
      work = work_of(a, seq);
    }
    const int64_t item = offset / work.units;
    const int from = static_cast<int>(offset - item * work.units);
    const int64_t left = end - done;
    const int to = static_cast<int>(left < work.units - from ? from + left : work.units);
    done += to - from;
    offset += to - from;
    g->seq = seq;
    g->s = s;
    if (a.split) {
      g->head = static_cast<int>(item / work.tiles);
      g->tile = static_cast<int>(item - static_cast<int64_t>(g->head) * work.tiles);
    } else {
      // the last tiles of all heads come first: they see the most keys
      const int64_t tile = item / a.pool.kv_heads;
      g->head = static_cast<int>(item - tile * a.pool.kv_heads);
      g->tile = work.tiles - 1 - static_cast<int>(tile);
    }
    const int t0 = static_cast<int>(static_cast<int64_t>(g->tile) * a.tile_rows / a.group);
    g->first_position = seq.length - seq.n + t0;
    g->lo = first_key(a, seq, a.split ? 0 : t0);
    g->hi = seq.length;
    if (a.split) {
      // (all tiles of a sequence go through the same units, so that they count the same)
      g->from = g->lo / kUnit + from;
      g->to = g->lo / kUnit + to;
    } else {
      const int64_t t1 = (static_cast<int64_t>(g->tile + 1) * a.tile_rows - 1) / a.group;
      g->hi = max(seq.length - seq.n + static_cast<int>(t1 < seq.n ? t1 + 1 : seq.n), 0);
      g->from = g->lo / kUnit;
      g->to = (g->hi + kUnit - 1) / kUnit;
    }
    // a block's first segment may continue an item, its last may be continued; one that is both is the first
    g->slot = from == 0 && to == work.units ? 0 : from > 0 ? 1 : 2;
    g->item = (static_cast<int64_t>(s) * a.pool.kv_heads + g->head) << 32 | g->tile;
    return true;
  }
};

// Every thread of the block: its share.  false: nothing to do (a split block then has marked its slots).
template <int THREADS>
__device__ bool share(const Attend& a, int64_t* shared, Share* r) {
  int64_t place = 0, last = 0;
  const int64_t block = blockIdx.x, blocks = gridDim.x;
  int s;
  int64_t offset;
  find_place<THREADS>(
      a, shared,
      [&](int64_t total) {
        // (with fewer units than blocks the first `total` blocks have one each)
        const int64_t n = a.split ? (total < blocks ? total : blocks) : total;
        place = !a.split ? block : block < n ? block * total / n : total;
        last = !a.split ? (block < total ? block + 1 : block) : block < n ? (block + 1) * total / n : total;
        return place;
      },
      &s, &offset);
  if (place >= last || s >= a.pool.sequences) {
    if (a.split && threadIdx.x < 2) a.slots[2 * block + threadIdx.x] = -1;
    return false;
  }
  r->begin = r->done = place;
  r->end = last;
  r->s = s;
  r->offset = offset;
  r->seq = sequence(a.pool, s);
  r->work = work_of(a, r->seq);
  return true;
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

// host side: each returns a status
constexpr int kMaxBlocks = 1024;  // of a split launch (the join kernel's table of weights)
int rows_tile(int dim);           // rows of an item in the CUDA-core kernel
int launch_rows(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream);
int token_blocks_per_sm(int cache_dtype, int dim);
constexpr int kTokenRows = 16;    // rows of an item in the 16- and 8-bit kernel
bool token_fits(const ksmm_cache_attention_desc_t& d);
int launch_token(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream);
int prompt_rows(int dim, int group);  // rows of an item in the prompt kernel
bool prompt_fits(const ksmm_cache_attention_desc_t& d);
int launch_prompt(const Attend& a, int dtype, unsigned grid, cudaStream_t stream);
int launch_join(const Attend& a, int dtype, unsigned blocks, cudaStream_t stream);

}  // namespace cache
}  // namespace ksmm
