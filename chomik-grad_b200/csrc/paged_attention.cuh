// Shared by the kernels of cb_paged_attention and cb_paged_attention_shared: the
// division of the work over a launch's blocks, and the results that several
// blocks join.
#pragma once

#include <climits>

#include "paged.cuh"
#include "sync.cuh"

namespace cb {

// The first keys of all sequences of a call, computed apart (paged_shared.cu).
// `common`: for each sequence the whole pages that it has in common with the
// call's first; INT_MAX where it takes no part.  The rows of a kv head, those
// of all sequences, go in blocks of `block_rows`; an item is a kv head and a block
// of rows, and its keys, in tiles of kSharedTile, are cut into `splits` pieces (see
// shared_cut).  Piece s of item i is parts (i * splits + s) * ways .. + ways - 1:
// references of block_rows rows, their sums, then the rows' elements (see shared_at).
constexpr int kSharedTile = 64;
struct SharedKeys {
  const int* common;  // and behind them the slot of the first sequence that takes part
  const float* parts;
  int block_rows, ways, blocks, least;  // blocks of the grid; tiles of a piece: `least` or more, or all
  long long least_bytes;                // of reads that are repeated; below 0: see worth_sharing
};
// Whether `keys` that `sequences` hold in common are computed apart.  Where the caller leaves
// it open, from 192 MB on that all but three of the sequences would read: beginning, ending
// and joining the parts takes 25 to 30 us, and a pass of the shared kernel about as long as
// three sequences' reads by the other one (8 kv heads of 128; apart and not: 64 sequences of
// one token, 1024 keys 42 us and 38, 2048 43 and 58, 16384 69 and 356; 16 of 5 tokens, 4400
// keys 66 and 53, 8192 77 and 82; 8 of one token, 8192 keys 43 and 33, 16384 51 and 53; 4, 65536
// keys 103 and 101; 2, 131072 keys 160 and 101).  And items for a 32nd of the SMs: of fewer
// each is cut in so many pieces that joining them takes longer than the reads (one kv head,
// 32 rows, 16 sequences of 65536 keys: 74 pieces, 191 us and 105).
constexpr int kSharedReads = 3, kSharedPieces = 32;
constexpr long long kSharedBytes = 192LL << 20;
__host__ __device__ inline bool worth_sharing(const cb_paged_attention_args& a, const SharedKeys& s, long long sequences,
                                              long long keys) {
  const long long each = keys * a.cache.kv_heads * a.cache.head_size * 2;
  if (s.least_bytes >= 0) return (sequences - 1) * each >= s.least_bytes;
  const long long rows = a.batch * a.tokens * (a.heads / a.cache.kv_heads);
  const long long items = a.cache.kv_heads * ((rows + s.block_rows - 1) / s.block_rows);
  return (sequences - kSharedReads) * each >= kSharedBytes && items * kSharedPieces >= s.blocks;
}
// Of element d of row r behind a part's references and sums: eight elements of all rows
// together, a sector each.
__host__ __device__ constexpr long long shared_at(int block_rows, int r, int d) {
  return (static_cast<long long>(d / 8) * block_rows + r) * 8 + d % 8;
}
// cb_paged_attention's launch, of the keys behind the shared ones where `shared` is given.
int launch_attention(const cb_paged_attention_args& a, const SharedKeys* shared, void* scratch, unsigned* counters,
                     cudaStream_t stream);
// Bytes of scratch that it needs.
long long attention_scratch(const cb_paged_attention_args& a, bool shared);

inline int attention_check(const cb_paged_attention_args& a, const char* who) {
  const int status = paged_cache_check(a.cache, who);
  if (status != CB_OK) return status;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "%s: q must be float32, bfloat16 or float16", who);
  CB_REQUIRE(a.heads >= 1 && a.heads <= (1 << 20) && a.heads % a.cache.kv_heads == 0,
             "%s: %lld heads for %d kv heads", who, a.heads, a.cache.kv_heads);
  CB_REQUIRE(a.batch >= 0 && a.batch <= 65535 && a.tokens >= 0 && a.tokens <= 65535 &&
                 a.tokens * (a.heads / a.cache.kv_heads) < (1LL << 30),
             "%s: %lld sequences of %lld tokens", who, a.batch, a.tokens);
  return CB_OK;
}

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

// Four codes -> two pairs of halves: of int8 elements 0, 2 and 1, 3, of e4m3
// elements 0, 1 and 2, 3.  int8: the byte x + 128 (the sign bit turned) under
// the exponent of 1024 is the number 1152 + x; one logic instruction makes two.  (The
// method: Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022.)
template <int STORAGE>
__device__ __forceinline__ void to_halves(uint32_t w, uint32_t& a, uint32_t& b) {
  if (STORAGE == CB_I8) {
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t even, odd;
    asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;" : "=r"(even) : "r"(w));  // (w & mask) ^ bits
    asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;" : "=r"(odd) : "r"(w >> 8));
    a = bits(__hsub2(*reinterpret_cast<const __half2*>(&even), bias));
    b = bits(__hsub2(*reinterpret_cast<const __half2*>(&odd), bias));
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
}
struct Plan {  // of one launch
  cb_paged_attention_args a;
  int group, rows, blocks;  // query heads of a kv head, rows of a kv head, blocks of them
  bool wide;                // queries can be read 16 bytes at a time
  float* partial;           // scratch: two partial results of each block
  unsigned* arrived;        // for each block: parts of the item that it begins and does not end
  SharedKeys shared;
};

// Pages that all sequences of the call have in common, 0 where it is not worth their
// being computed apart; every thread of the block calls this.
__device__ __forceinline__ int common_pages(const cb_paged_attention_args& a, const SharedKeys& shared, int* found) {
  if (threadIdx.x == 0) {
    found[0] = INT_MAX;
    found[1] = 0;
  }
  __syncthreads();
  int least = INT_MAX, there = 0;
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
    const int pages = __ldcg(shared.common + b);
    least = min(least, pages);
    there += pages != INT_MAX;
  }
  least = __reduce_min_sync(0xffffffffu, least);
  there = __reduce_add_sync(0xffffffffu, there);
  if ((threadIdx.x & 31) == 0 && there > 0) {
    atomicMin(found, least);
    atomicAdd(found + 1, there);
  }
  __syncthreads();
  if (found[1] == 0) return 0;
  const long long keys = static_cast<long long>(found[0]) * a.cache.page;
  return worth_sharing(a, shared, found[1], keys) ? found[0] : 0;
}
// The division of the shared keys: tiles of an item and of a piece, pieces of an item.
// No block takes pieces of two items while there are more blocks than items, since
// beginning and ending one takes as long as several tiles.
struct SharedCut {
  int tiles, per, splits;
};
__device__ __forceinline__ SharedCut shared_cut(const SharedKeys& s, int items, int keys) {
  SharedCut cut;
  cut.tiles = (keys + kSharedTile - 1) / kSharedTile;
  const int splits = max(1, min(s.blocks / items, (cut.tiles + s.least - 1) / s.least));
  cut.per = (cut.tiles + splits - 1) / splits;
  cut.splits = cut.per > 0 ? (cut.tiles + cut.per - 1) / cut.per : 1;
  return cut;
}

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
// `skip`: columns of the table that are left out (at least one key of each row is not among them).
template <int TILE>
__device__ __forceinline__ Slot slot_of(const Plan& p, long long b, int skip) {
  Slot s;
  if (!paged_row(p.a.cache, p.a.sequences, p.a.counts, p.a.tokens, b, p.a.error_flag, &s.row)) {
    s.row.length = s.row.count = 0;
    s.row.table = p.a.cache.table;
  }
  if (s.row.count > 0) {
    s.row.table += skip;
    s.row.length -= skip * p.a.cache.page;
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
  int b, origin, at, range, end, per, items, skip;

  __device__ __forceinline__ bool next(const Plan& p, Segment* g) {
    while (at < end) {
      int span = s.tiles + kItemCost;
      if (at - origin >= span * items) {
        origin += span * items;
        s = slot_of<TILE>(p, ++b, skip);
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
__device__ __forceinline__ bool begin_walk(const Plan& p, int skip, int* scan, int* found, Walk<TILE>* walk) {
  constexpr int kBlock = 32 * WARPS;
  const int batch = static_cast<int>(p.a.batch), items = p.a.cache.kv_heads * p.blocks;
  Slot s;
  s.tiles = -kItemCost;
  int mine = 0, all;
  for (int b = batch - 1 - (batch - 1 - static_cast<int>(threadIdx.x)) % kBlock; b >= 0 && b < batch; b -= kBlock) {
    s = slot_of<TILE>(p, b, skip);  // (slot threadIdx.x last)
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
      if (b < batch) s = slot_of<TILE>(p, b, skip);
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
  walk->s.row.table = p.a.cache.table + found[2] * p.a.cache.columns + (found[4] > 0 ? skip : 0);
  walk->s.row.length = found[3];
  walk->s.row.count = found[4];
  walk->s.tiles = tiles_of<TILE>(walk->s.row);
  walk->at = walk->range = range;
  walk->end = end;
  walk->per = per;
  walk->items = items;
  walk->skip = skip;
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

// Weighted values v of a row's elements d .. d + 3 and the sum of its weights
// against the reference `top`, with those of the shared keys added in the order of
// the ranges.  `row` counts those of the kv head in all sequences.
template <int SIZE>
__device__ __noinline__ void add_shared(const Plan& p, int pages, long long row, int head, int d, float* top_,
                                        float* sum_, float* v) {
  const SharedKeys& s = p.shared;
  const int blocks = static_cast<int>((p.a.batch * p.rows + s.block_rows - 1) / s.block_rows);
  const SharedCut cut = shared_cut(s, p.a.cache.kv_heads * blocks, pages * p.a.cache.page);
  const int item = head * blocks + static_cast<int>(row / s.block_rows), r = static_cast<int>(row % s.block_rows);
  const long long floats = static_cast<long long>(s.block_rows) * (SIZE + 2);
  const float* parts = s.parts + static_cast<long long>(item) * cut.splits * s.ways * floats;
  const int count = cut.splits * s.ways;
  float top = *top_, sum = *sum_;
  constexpr int kBatch = 8;  // parts whose loads are in flight together
  for (int at = 0; at < count; at += kBatch) {
    float m[kBatch], l[kBatch], now = top;
    float4 x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float* part = parts + (at + k) * floats;
      m[k] = at + k < count ? __ldcg(part + r) : -INFINITY;
      l[k] = at + k < count ? __ldcg(part + s.block_rows + r) : 0.0f;
      x[k] = at + k < count
                 ? __ldcg(reinterpret_cast<const float4*>(part + 2 * s.block_rows + shared_at(s.block_rows, r, d)))
                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) now = fmaxf(now, m[k]);
    if (now == -INFINITY) continue;  // nothing yet
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
  *top_ = top;
  *sum_ = sum;
}

// An item that a cut divided: its first part, then the first partial results of
// the following blocks (`rest` + 2 k of them), in that order.
template <int SIZE, int ROWS, bool SHARED>
__device__ __noinline__ void join(const Plan& p, long long b, int head, int first_row, int count, int parts,
                                  const float* first, const float* rest, int pages, int thread, int threads) {
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
    if (SHARED && pages > 0 && row / p.group < count) add_shared<SIZE>(p, pages, b * p.rows + row, head, d, &top, &sum, v);
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
