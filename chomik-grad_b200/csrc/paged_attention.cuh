// Shared by the kernels of cb_paged_attention: the division of the work over a
// launch's blocks, and the results that several blocks join.
#pragma once

#include "paged.cuh"
#include "sync.cuh"

namespace cb {
namespace {

// Tiles' time that beginning an item costs (queries, first loads, joining the
// warps): counted when the work is divided.  2 / 3 / 4 / 5: a ragged batch 39.3
// / 39.2 / 39.0 / 40.0 us, drafted blocks 70.5 / 70.2 / 69.5 / 68.5.
constexpr int kItemCost = 4;
// Items of no more than six tiles are not cut: joining parts takes as long.
constexpr int kSmallItem = kItemCost + 6;

// 2^x by the hardware's instruction: its relative error is below 2^-22, and
// results below 2^-126 are zero (weights are at most one).
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x as the square of this: a sum may be large enough that its share is
// kept where 2^x itself would be below float32's range.
__device__ __forceinline__ float root2_of(float x) { return exp2_of(0.5f * x); }

// Value scales are taken against 2^base, twice the power of two of the first that
// is not zero.  One from 2^-kScales of it to less than twice goes into the weights as it is; others
// leave their exponent e, against base, to the score, and 2^-e to the weight's
// share in the sum of the weights.  From -kZeroBelow (which zeros count as: they
// belong to that sum alone) to kMostAbove both sums stay within float32; a larger
// scale moves base, and of that up to kMostLower the scores' reference, the rest
// the weighted values.
constexpr int kScales = 5, kZeroBelow = 64, kMostAbove = 100, kMostLower = 24, kLeastField = 7;
constexpr uint32_t kNoScale = 0xfc000000u;  // (of no scale but those below -2^121)

// The sums are kept against a reference c: a score x, its scale's exponent
// included, weighs 2^(x - c), and 2^kLift times that in fp16.  A step whose
// largest x is more than kWindow from c moves c to kAbove below it, up or down
// (by an even number: sums move by exact powers of two).  So the largest weight
// of a step, with a scale like the first, lies between 2^-7 and 2^15, where two
// fp16 parts hold it to 18 bits at worst and to 22 in the upper half, and the
// step's others to 2^-25: keys far below one that was seen before keep their
// bits, and only those that share their step of 2048 / head_size keys with a far
// heavier one are off, by up to 2^-30 of its weight each.  Down by at most kDown
// at a time, and not where the sums would come near float32's end.
constexpr float kWindow = 10.0f, kAbove = 4.0f, kDown = 50.0f, kUnset = -1e30f;
constexpr int kLift = 4, kRoom = 20;

// 2^e, e in [-126, 127]
__device__ __forceinline__ float power2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

struct Plan {  // of one launch
  cb_paged_attention_args a;
  int group, rows, blocks;  // query heads of a kv head, rows of a kv head, blocks of them
  bool wide;                // queries can be read 16 bytes at a time
  float* partial;           // scratch: two partial results of each block
  unsigned* arrived;        // for each block: parts of the item that it begins and does not end
};

inline Plan plan_of(const cb_paged_attention_args& a, int block_rows, void* scratch, unsigned* counters) {
  Plan p;
  p.a = a;
  p.group = static_cast<int>(a.heads / a.cache.kv_heads);
  p.rows = static_cast<int>(a.tokens * p.group);
  p.blocks = (p.rows + block_rows - 1) / block_rows;
  const int item = a.dtype == CB_F32 ? 4 : 2;
  p.wide = reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
  for (int i = 0; i < 3; ++i) p.wide = p.wide && a.q_strides[i] * item % 16 == 0;
  p.partial = static_cast<float*>(scratch);
  p.arrived = counters;
  return p;
}

// Blocks that fill the GPU once, and no more than there can be tiles; 0 where a
// launch could have more units of work than can be divided in 32 bits (they are
// rounded up to a multiple of the blocks).
inline long long grid_of(const cb_paged_attention_args& a, int block_rows, int tile, int per_sm) {
  const long long rows = a.tokens * (a.heads / a.cache.kv_heads), blocks = (rows + block_rows - 1) / block_rows;
  const long long tiles = (a.cache.columns * a.cache.page + tile - 1) / tile;
  const double most = static_cast<double>(a.batch) * a.cache.kv_heads * blocks * (tiles + kItemCost);
  const long long fill = 1LL * per_sm * sm_count();
  if (most + static_cast<double>(fill) >= 2147483648.0) return 0;
  return most < fill ? static_cast<long long>(most) : fill;
}

struct Slot {
  PagedRow row;
  int tiles;
};
template <int TILE>
__device__ __forceinline__ int tiles_of(const PagedRow& row) {
  const int keys = row.count > 0 ? row.length : 1;  // (an item without keys writes zeros)
  return (keys - 1) / TILE + 1;                     // (no sum that passes 2^31)
}
template <int TILE>
__device__ __forceinline__ Slot slot_of(const Plan& p, long long b) {
  Slot s;
  if (!paged_row(p.a.cache, p.a.sequences, p.a.counts, p.a.tokens, b, p.a.error_flag, &s.row)) {
    s.row.length = s.row.count = 0;
    s.row.table = p.a.cache.table;
  }
  s.tiles = tiles_of<TILE>(s.row);
  return s;
}

template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int* shared, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w == warp) before = all;
    all += shared[w];
  }
  *total = all;
  return before + incl - v;
}

// A run of tiles of one item (slot, kv head, block of rows) that a block takes.
struct Segment {
  Slot s;
  int b, item, tile, tiles;
  bool whole, begins;  // all of the item; its first tile is the first of the block's range
  int from, last;      // blocks that hold the item's first and last tile, where it is cut
  bool from_begins;    // `begins` of the first of them
  bool empty;          // no rows: the result is zeros
};

// The segments of one block, in order.  The units of all items, kItemCost of
// each item's own and then its tiles, are cut in equal ranges.
template <int TILE>
struct Walk {
  Slot s;
  int b, origin, at, range, end, per, items;

  __device__ __forceinline__ bool next(const Plan& p, Segment* g) {
    while (at < end) {
      int span = s.tiles + kItemCost;
      if (at - origin >= span * items) {
        origin += span * items;
        s = slot_of<TILE>(p, ++b);
        span = s.tiles + kItemCost;
      }
      const int item = (at - origin) / span, item_at = origin + item * span;
      const bool small = span <= kSmallItem;  // belongs to the block in whose range it begins
      g->tile = max(0, at - item_at - kItemCost);
      g->tiles = small ? (at == item_at ? s.tiles : 0) : max(0, min(end - item_at, span) - kItemCost) - g->tile;
      at = item_at + span;
      if (g->tiles <= 0) continue;
      g->s = s;
      g->b = b;
      g->item = item;
      g->whole = g->tile == 0 && g->tiles == s.tiles;
      g->begins = item_at + kItemCost <= range;
      g->from = (item_at + kItemCost) / per;
      g->last = (item_at + span - 1) / per;
      g->from_begins = item_at + kItemCost <= g->from * per;
      g->empty = s.row.count == 0;
      return true;
    }
    return false;
  }
};

// Finds the block's range; every thread of it calls this.  False: none.
template <int TILE, int WARPS>
__device__ __forceinline__ bool begin_walk(const Plan& p, int* scan, int* found, Walk<TILE>* walk) {
  constexpr int kBlock = 32 * WARPS;
  const int batch = static_cast<int>(p.a.batch), items = p.a.cache.kv_heads * p.blocks;
  Slot s;
  s.tiles = -kItemCost;
  int mine = 0, all;
  for (int b = batch - 1 - (batch - 1 - static_cast<int>(threadIdx.x)) % kBlock; b >= 0 && b < batch; b -= kBlock) {
    s = slot_of<TILE>(p, b);  // (slot threadIdx.x last)
    mine += s.tiles + kItemCost;
  }
  block_scan<WARPS>(mine, scan, &all);
  all *= items;
  const int per = (all + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int range = per * static_cast<int>(blockIdx.x), end = min(range + per, all);
  if (range >= end) return false;
  int before = 0;
  for (int first = 0; first < batch; first += kBlock) {
    const int b = first + static_cast<int>(threadIdx.x);
    if (first > 0) {
      if (b < batch) s = slot_of<TILE>(p, b);
      else s.tiles = -kItemCost;
    }
    const int units = (s.tiles + kItemCost) * items;
    int sum;
    const int lower = before + block_scan<WARPS>(units, scan, &sum);
    if (lower <= range && range < lower + units) {
      found[0] = b;
      found[1] = lower;
      found[2] = static_cast<int>((s.row.table - p.a.cache.table) / p.a.cache.columns);
      found[3] = s.row.length;
      found[4] = s.row.count;
    }
    before += sum;
    if (before > range) break;
  }
  __syncthreads();
  walk->b = found[0];
  walk->origin = found[1];
  walk->s.row.table = p.a.cache.table + found[2] * p.a.cache.columns;
  walk->s.row.length = found[3];
  walk->s.row.count = found[4];
  walk->s.tiles = tiles_of<TILE>(walk->s.row);
  walk->at = walk->range = range;
  walk->end = end;
  walk->per = per;
  walk->items = items;
  return true;
}

// Eight neighbouring elements of a query row.
__device__ __forceinline__ void load_query(const Plan& p, const void* query, long long at, float* x) {
  if (!p.wide) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_as_f32(query, at + i, p.a.dtype);
  } else if (p.a.dtype == CB_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(query) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(query) + at + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(query) + at);
    if (p.a.dtype == CB_BF16) {
      unpack_bf16x8(w, x);
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __low2float(h[i]);
        x[2 * i + 1] = __high2float(h[i]);
      }
    }
  }
}

// Where row r of an item goes; r past the item's rows: nowhere.
template <int SIZE>
__device__ __forceinline__ long long out_row(const Plan& p, long long b, int head, int r) {
  return ((b * p.a.tokens + r / p.group) * p.a.heads + head * p.group + r % p.group) * SIZE;
}
__device__ __forceinline__ void store4(const Plan& p, long long at, const float* v) {
  if (p.a.dtype == CB_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint2 w;
    if (p.a.dtype == CB_BF16) {
      __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      w = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    } else {
      w = make_uint2(bits(__floats2half2_rn(v[0], v[1])), bits(__floats2half2_rn(v[2], v[3])));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.a.out) + at) = w;
  }
}

// Partial results: maxima and sums of the rows, then the rows.
__host__ __device__ constexpr int partial_floats(int size, int rows) { return rows * (size + 2); }

// An item that a cut divided: its first part, then the first partial results of
// the following blocks (`rest` + 2 k of them), in that order.
template <int SIZE, int ROWS>
__device__ __noinline__ void join(const Plan& p, long long b, int head, int first_row, int count, int parts,
                                  const float* first, const float* rest, int thread, int threads) {
  constexpr int kRows = ROWS, kFloats = partial_floats(SIZE, ROWS);
  for (int i = thread; i < kRows * SIZE / 4; i += threads) {
    const int r = i / (SIZE / 4), d = i % (SIZE / 4) * 4, row = first_row + r;
    if (row >= p.rows) continue;
    float top = -INFINITY, sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kBatch = 8;  // parts whose loads are in flight together
    for (int from = 0; from < parts; from += kBatch) {
      float m[kBatch], l[kBatch], now = top;
      float4 x[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int at = from + k;
        const float* part = at ? rest + 2LL * at * kFloats : first;
        m[k] = at < parts ? __ldcg(part + r) : -INFINITY;
        l[k] = at < parts ? __ldcg(part + kRows + r) : 0.0f;
        x[k] = at < parts ? __ldcg(reinterpret_cast<const float4*>(part + 2 * kRows + r * SIZE + d))
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) now = fmaxf(now, m[k]);
      const float keep = top == -INFINITY ? 0.0f : root2_of(top - now);
      sum = sum * keep * keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = v[i] * keep * keep;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float f = m[k] == -INFINITY ? 0.0f : root2_of(m[k] - now);
        sum += f * l[k] * f;
        v[0] += f * x[k].x * f; v[1] += f * x[k].y * f; v[2] += f * x[k].z * f; v[3] += f * x[k].w * f;
      }
      top = now;
    }
    const bool real = row / p.group < count && sum != 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = real ? v[k] / sum : 0.0f;
    store4(p, out_row<SIZE>(p, b, head, row) + d, v);
  }
}

// This block's part of a cut item is written (by every thread before the
// caller's barrier): whether it was the last, which joins them.  One thread calls.
__device__ __forceinline__ bool last_part(const Plan& p, const Segment& g) {
  const bool last = ticket_acq_rel(p.arrived + g.from) == static_cast<unsigned>(g.last - g.from);
  if (last) p.arrived[g.from] = 0;
  return last;
}
template <int SIZE, int ROWS>
__device__ __forceinline__ float* part_of(const Plan& p, int block, bool begins) {
  return p.partial + (2LL * block + (begins ? 0 : 1)) * partial_floats(SIZE, ROWS);
}

}  // namespace
}  // namespace cb
