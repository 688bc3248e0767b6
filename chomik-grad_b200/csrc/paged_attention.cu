// Attention over the paged 8-bit KV cache: cb_paged_attention.
//
// For the query row of token t of the last n of a slot with `length` keys,
// head h of kv head g = h / (heads / kv_heads):
//   s_j = scale * ks[page(j), g] * sum_d q_d kq[j, d],  j <= length - n + t
//   out = sum_j exp(s_j - m) vs[page(j), g] vq[j, :] / sum_j exp(s_j - m)
//
// What bounds it: the cache is read once, 2 * head_size bytes a key and kv
// head, for 2 flops a byte and query row.  The rows that share a kv head
// (tokens * heads / kv_heads of them) are multiplied together, so that the
// bytes stay the bound up to about 32 rows; with 8 rows the multiply-adds
// alone (184 a clock and SM at the measured 6.47 TB/s) are beyond the FP32
// units, so the products go to the tensor cores as fp16 m16n8k16 products
// with float32 sums:
//   - int8 and e4m3 codes are exact in fp16, and the scales stay outside the
//     products: one factor for each 16 keys, since a page is 16 tokens or more;
//   - a query row is scaled by a power of two to below 2 and split into
//     hi + lo (22 bits); up to 8 rows, the hi parts are rows 0-7 of the tile
//     and the lo parts rows 8-15, at no cost.  16-bit queries in more than 8
//     rows take the hi part alone (exact but for elements 2^-14 below the row's
//     largest, whose error is below 2^-25 of that);
//   - what multiplies the value codes is the weight 2^(x - c) times the page's
//     value scale, both against references that follow the keys (see
//     paged_attention.cuh), so that these products stay within fp16 and keep their
//     bits however far apart scores and scales are.  They are split the same way
//     (bfloat16 outputs of more than 8 rows: hi only, a relative error of 2^-12 a
//     weight, a sixteenth of the output's own rounding; float16 outputs keep both,
//     for an error of 2.1e-4 against 2.9e-4 and 9 us of 69 in blocks of 20 rows).
//     The sum of the weights leaves the scale out.
//
// How the work is laid out.  The keys of all (slot, kv head, block of rows)
// are one sequence of tiles, cut into equal ranges for a grid that fills the
// GPU once, whatever the lengths: each block finds its range from the lengths
// on the device.  An item that a cut divides leaves partial results (reference,
// sum, weighted values), which the block that finishes last joins in the order
// of the keys: equal inputs give equal bits, and there is one launch.
//
// Within a tile each warp takes its own 16, 32 or 64 keys (4 KB for any head
// size) with references of its own, joined at the end of an item: no
// block barrier inside the loop.  A warp copies its keys through shared memory
// with 16-byte asynchronous copies, one to three steps ahead; keys beyond the
// length are filled with zeros, whatever the page holds there.
//
// Measured, one B200, 8 kv heads of 128: two sequences of 131,067 keys, e4m3,
// 4 rows: 94.5 us, 5.7 TB/s (88% of the measured copy); 32 ragged sequences of up
// to 4096, int8, 4 rows: 39.5 us, 4.1 TB/s (3 us until the first products, 5.7
// TB/s after that, blocks' ends 28 to 41 us apart by their share of begins,
// ends and joins); 16 ragged ones of up to 8191, int8, float16, 20 rows: 69 to 72
// us by where the pool lies in memory, 2.4 TB/s, where 8 warps an SM leave the
// latency of the instructions open (IPC 1.67, tensor pipe 40%).  One sequence of
// 384 keys: 7.4 us of dependent loads.  References that follow scores and scales
// cost 0.4 us of these at the long ones, 0.9 at the batch, 3 in the drafted blocks.
#include <type_traits>

#include "paged_attention.cuh"

namespace cb {
namespace {

constexpr int kGroups = 4;                       // of keys, in a tile
constexpr int kStepBytes = 4096;                 // K and V of a group's step
constexpr int kHeadBytes = 64;                   // its scales: 4 of K, 4 of V
constexpr int kSlotBytes = kStepBytes + kHeadBytes;

// MODE is the number of 8-row sets that a block takes: one set with both parts
// in one 16-row tile of the scores' products, or two to four, two to a tile.
enum { kPacked = 1 };
// Low parts of unpacked rows: none (bfloat16), of queries and weights (float32),
// of the weights alone (float16, whose queries are exact).
enum { kNoParts = 0, kBothParts = 1, kWeightParts = 2 };
__host__ __device__ constexpr int tiles_of_mode(int mode) { return (mode + 1) / 2; }
__host__ __device__ constexpr int rows_of(int mode) { return 8 * mode; }
constexpr int kThreads = 32 * kGroups;
// Resident blocks of an SM by the registers of a warp's sums: 12 warps of 168
// for one set (its queries stay in registers too: 97 us against 102 with 16
// warps at two sequences of 131,067 keys, 8 kv heads of 128) and two (47 us
// against 53 with 16 warps that spill, 12 rows, 16 x 5100 keys on average,
// bfloat16), 8 of 255 for three and four (62 against 70 with 12 warps, 20 rows).
// The steps of a warp's ring: as few as the join at an item's end leaves (two
// against four: 94 us and 97 at the long sequences, 45.6 and 47.4 with 12 rows;
// 8 KB a warp in flight are 96 KB an SM).
__host__ __device__ constexpr int resident_of(int mode) {
  return mode >= 3 ? 2 : 3;
}
__host__ __device__ constexpr int stages_of(int mode) {
  return mode == 4 ? 4 : mode == 3 ? 3 : 2;
}
__host__ __device__ constexpr int ring_bytes(int mode) { return kGroups * stages_of(mode) * kSlotBytes; }
__host__ __device__ constexpr int step_keys(int head_size) { return 2048 / head_size; }
__host__ __device__ constexpr int tile_keys(int head_size) { return kGroups * step_keys(head_size); }

// Shared memory of a block: the ring, and the queries as the products read them.
__host__ __device__ constexpr int shared_bytes(int head_size, int mode, int lo) {
  return ring_bytes(mode) + tiles_of_mode(mode) * (lo == kBothParts ? 2 : 1) * (head_size / 16) * 512;
}

// ---- loads -------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_of(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_groups() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte piece `piece` of row `row` in a buffer of rows of
// SIZE bytes.  The 16-byte places of a 128-byte line are exchanged by the
// line's number so that the reads below touch every bank once.
template <int SIZE>
__device__ __forceinline__ int swizzled(int row, int piece) {
  const int at = row * (SIZE / 16) + piece, line = at >> 3;
  const int turn = SIZE == 128 ? line & 7 : SIZE == 64 ? (line & 1) | ((line & 2) << 1) : (line & 1) << 2;
  return (line << 7) + (((at & 7) ^ turn) << 4);
}
// Key of column n of an 8-key tile, and the first of the SIZE / 8 elements of
// column n of the value tiles: the orders are free, and these go with `swizzled`.
__device__ __forceinline__ int key_of(int n) { return (n >> 1) + (n & 1) * 4; }
template <int SIZE>
__device__ __forceinline__ int element_of(int n) {
  if (SIZE == 128) return (((n & 1) << 2) | (n >> 1)) * 16;
  if (SIZE == 64) return ((n >> 2) + ((n >> 1) & 1) * 2) * 16 + (n & 1) * 8;
  return n * 4;
}

template <int WORDS>
__device__ __forceinline__ void read_words(const char* p, uint32_t* w) {
  if (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// ---- fp16 operands -------------------------------------------------------------

// The words whose pairs are elements 2 i and 2 i + 1 of two rows, i = 0, 1.
template <int STORAGE>
__device__ __forceinline__ uint32_t interleave(uint32_t a, uint32_t b, int i) {
  if (STORAGE == CB_I8) return __byte_perm(a, b, i ? 0x7632 : 0x5410);
  return __byte_perm(a, b, i ? 0x7362 : 0x5140);
}

__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  hi = bits(h);
  lo = bits(__floats2half2_rn(x - __low2float(h), y - __high2float(h)));
}

// c (+)= a b; FIRST: from zero.
template <bool FIRST>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (FIRST) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// ---- one item ------------------------------------------------------------------

// The sums of one warp, g = lane / 4, c = lane % 4.  The maximum and the sum of
// the weights are those of row g of each 8-row set.  The weighted values are
// computed transposed, value elements as the products' 16 rows and the set as
// their 8 columns: no row of a product is wasted, and the weights are its second
// operand as the scores' products leave them.  o[set][j] holds elements 2 j (the
// first two) and 2 j + 1 of column element_of(g), for rows 2 c and 2 c + 1.
template <int SIZE, int MODE>
struct Sums {
  static constexpr int kTiles = tiles_of_mode(MODE);
  float o[MODE][SIZE / 16][4];
  float m[MODE], l[MODE];
};

// The block's query rows as the products read them: `queries` holds the 16-row
// operands of each 16-element product, `factors` what turns a row's products
// into scores in base 2.  SIZE / 8 neighbouring threads take a row; rows that
// do not exist are zero.
template <int SIZE, int STORAGE, int MODE, int LO>
__device__ __forceinline__ void load_queries(const Plan& p, const void* query, int count, int head, int first_row,
                                             uint4* queries, float* factors) {
  constexpr int kLanes = SIZE / 8, kDots = SIZE / 16, kParts = LO == kBothParts ? 2 : 1;
  constexpr int kKeyWords = SIZE / 16 < 4 ? SIZE / 16 : 4;
  constexpr int kAll = MODE == kPacked ? 8 : 16 * tiles_of_mode(MODE);  // rows of the operands
#pragma unroll
  for (int first = 0; first < kAll; first += kThreads / kLanes) {
    const int row = first + static_cast<int>(threadIdx.x) / kLanes, d = static_cast<int>(threadIdx.x) % kLanes * 8;
    const int r = first_row + row, t = r / p.group;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, largest = 0.0f;
    if (row < rows_of(MODE) && r < p.rows && t < count)
      load_query(p, query, t * p.a.q_strides[1] + (head * p.group + r % p.group) * p.a.q_strides[2] + d, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    if (row >= kAll) continue;
    // 2^e <= largest < 2^(e + 1); e in [-126, 127], and 2^-e is exact
    const int e = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -126), 127);
    const float down = e == 127 ? 5.877471754111438e-39f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    if (d == 0 && row < rows_of(MODE))
      factors[row] = p.a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int word = 0; word < 2; ++word) {
      const int at = d + 4 * word;  // of word `k` of read at / 64 of a key row, by the lanes of column `quad`
      const int quad = at % 64 / (4 * kKeyWords), dot = at / 64 * kKeyWords + at % (4 * kKeyWords) / 4;
      uint32_t* to = reinterpret_cast<uint32_t*>(queries + (row / 16 * kParts * kDots + dot) * 32 + row % 8 * 4 + quad);
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        uint32_t hi, lo;
        const int first = 4 * word + (STORAGE == CB_I8 ? pair : 2 * pair), next = STORAGE == CB_I8 ? 2 : 1;
        split(x[first] * down, x[first + next] * down, hi, lo);  // in the pairs of to_halves
        if (MODE == kPacked) {
          to[2 * pair] = hi;
          to[2 * pair + 1] = lo;
        } else {
          to[2 * pair + row / 8 % 2] = hi;
          if (LO == kBothParts) to[kDots * 128 + 2 * pair + row / 8 % 2] = lo;
        }
      }
    }
  }
}

template <int SIZE, int STORAGE, int MODE, int LO>
__device__ __forceinline__ void warp_item(const Plan& p, const void* query, const Slot& s, int head, int first_row,
                                          int tile, int tiles, char* shared, float* factors,
                                          Sums<SIZE, MODE>& sums) {
  using S = Sums<SIZE, MODE>;
  constexpr int kKeys = step_keys(SIZE), kSubs = kKeys / 16, kStages = stages_of(MODE);
  constexpr int kDots = SIZE / 16;                          // 16-element products of a score
  constexpr int kKeyWords = SIZE / 16 < 4 ? SIZE / 16 : 4;  // words of one read of a key row
  constexpr int kKeyReads = SIZE / 16 / kKeyWords;
  constexpr int kValueWords = SIZE / 32;
  constexpr int kParts = LO == kBothParts ? 2 : 1;          // of the queries
  constexpr int kWeights = MODE == kPacked || LO ? 2 : 1;   // parts of the weights
  const cb_paged_cache& c = p.a.cache;
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
  char* ring = shared + group * kStages * kSlotBytes;
  uint4* queries = reinterpret_cast<uint4*>(shared + ring_bytes(MODE));

  // limits: row r sees keys below limit[r]; all rows of the warp see those below `common`
  int limit[MODE];
#pragma unroll
  for (int at = 0; at < MODE; ++at) {
    const int r = first_row + at * 8 + g, t = r / p.group;
    limit[at] = r < p.rows && t < s.row.count ? s.row.length - s.row.count + t + 1 : 0;
    sums.m[at] = kUnset;
    sums.l[at] = 0.0f;
#pragma unroll
    for (int j = 0; j < SIZE / 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums.o[at][j][i] = 0.0f;
  }
  uint32_t least = kNoScale;  // bits of 2^(base - kScales), once there is a scale
  float unit = 1.0f;          // 2^(kLift - base)
  int far = 0;                // the largest scale's exponent, where it is above base
  const int common = s.row.length - s.row.count + first_row / p.group + 1;
  const int length = s.row.length;

  // page ids: lane i of a batch holds that of the group's 16-key piece 32 * batch + i
  const int shift = 31 - __clz(c.page);
  auto piece_key = [&](int piece) {
    return (tile + piece / kSubs) * tile_keys(SIZE) + group * kKeys + (piece % kSubs) * 16;
  };
  auto ids_of = [&](int batch) {
    const int piece = batch * 32 + lane;
    if (piece >= tiles * kSubs) return -1;
    const int key = piece_key(piece);
    if (key >= length) return -1;
    const int page = s.row.table[key >> shift];
    if (page < 0 || page >= c.pages) {
      raise_flag(p.a.error_flag, CB_FLAG_BOOK);
      return -1;
    }
    return page;
  };
  int ids = ids_of(0), ids_next = ids_of(1), batch = 0;

  // A step is four copies of 32 x 16 bytes of K and four of V, 512 bytes apart;
  // odd ones of 128-byte rows are turned by half a line.
  constexpr int kRowCopies = SIZE / 32;  // of 16 rows
  const uint32_t page_bytes = static_cast<uint32_t>(c.kv_heads) * c.page * SIZE;
  const long long head_at = static_cast<long long>(head) * c.page * SIZE + lane * 16;
  const char* k_pool = static_cast<const char*>(c.k_pages) + head_at;
  const char* v_pool = static_cast<const char*>(c.v_pages) + head_at;
  const float* scale_of = (lane & 1 ? c.v_scale : c.k_scale) + head;
  const uint32_t scale_to = kStepBytes + (lane & 1 ? 16 : 0);
  const uint32_t to = swizzled<SIZE>(lane / (SIZE / 16), lane % (SIZE / 16));
  const uint32_t ring_at = shared_of(ring);
  uint32_t fill = ring_at;  // slot that is filled next
  auto prefetch = [&](int step) {
    if (step < tiles) {
      if (step * kSubs / 32 > batch) {
        ids = ids_next;
        ids_next = ids_of(++batch + 1);
      }
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const int piece = step * kSubs + sub, key = piece_key(piece);
        const int page = __shfl_sync(0xffffffffu, ids, piece & 31);
        const int rows = page >= 0 ? length - key : 0;  // that exist
        const long long from = static_cast<long long>(max(page, 0)) * page_bytes + (key & (c.page - 1)) * SIZE;
        const char *k = k_pool + from, *v = v_pool + from;
#pragma unroll
        for (int n = 0; n < kRowCopies; ++n) {
          const uint32_t dst = fill + ((SIZE == 128 && (n & 1) ? to ^ 64 : to) + (sub * kRowCopies + n) * 512);
          if (rows >= 16) {
            copy16(dst, k + n * 512);
            copy16(dst + 2048, v + n * 512);
          } else {
            const bool real = (n * 512 + lane * 16) / SIZE < rows;
            copy16(dst, k + n * 512, real);
            copy16(dst + 2048, v + n * 512, real);
          }
        }
        if (lane < 2)
          copy4(fill + scale_to + sub * 4, scale_of + static_cast<long long>(max(page, 0)) * c.kv_heads, page >= 0);
      }
    }
    commit();
    fill = fill + kSlotBytes == ring_at + kStages * kSlotBytes ? ring_at : fill + kSlotBytes;
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) prefetch(i);

  load_queries<SIZE, STORAGE, MODE, LO>(p, query, s.row.count, head, first_row, queries, factors);
  __syncthreads();
  float factor[MODE];
#pragma unroll
  for (int at = 0; at < MODE; ++at) factor[at] = factors[at * 8 + g];
  queries += lane;
  uint4 held[MODE == kPacked ? kDots : 1];  // packed queries stay in registers
#pragma unroll
  for (int dot = 0; dot < (MODE == kPacked ? kDots : 0); ++dot) held[dot] = queries[dot * 32];
  // where this lane reads: rows 8 n + key_of(g) of K, quad + 4 i of V.  The
  // second half of a 128-byte key row, and every other row of V, lie half a line
  // turned; the rest are constant distances.
  const int key_at = swizzled<SIZE>(key_of(g), quad * kKeyWords / 4) + quad * kKeyWords * 4 % 16;
  const int value_at = 2048 + swizzled<SIZE>(quad, element_of<SIZE>(g) / 16) + element_of<SIZE>(g) % 16;
  const char* slot = ring;
  for (int step = 0; step < tiles; ++step) {
    wait_groups<kStages - 2>();
    __syncwarp();  // all copies of this step have landed; all lanes have left the slot filled next
    prefetch(step + kStages - 1);
    if (step > 0) slot = slot + kSlotBytes == ring + kStages * kSlotBytes ? ring : slot + kSlotBytes;
    const int key = (tile + step) * tile_keys(SIZE) + group * kKeys;
    const float* scales = reinterpret_cast<const float*>(slot + kStepBytes);

    float score[S::kTiles][2 * kSubs][4];
#pragma unroll
    for (int r = 0; r < kKeyReads; ++r) {
      uint32_t w[2 * kSubs][kKeyWords];
      const char* row = slot + (key_at ^ (r * 64));
#pragma unroll
      for (int n = 0; n < 2 * kSubs; ++n) read_words<kKeyWords>(row + n * 8 * SIZE, w[n]);
#pragma unroll
      for (int k = 0; k < kKeyWords; ++k) {
        const int dot = r * kKeyWords + k;
        uint4 a[S::kTiles][kParts];
#pragma unroll
        for (int mt = 0; mt < S::kTiles; ++mt)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            a[mt][part] = MODE == kPacked ? held[dot] : queries[((mt * kParts + part) * kDots + dot) * 32];
#pragma unroll
        for (int n = 0; n < 2 * kSubs; ++n) {
          uint32_t b0, b1;
          to_halves<STORAGE>(w[n][k], b0, b1);
#pragma unroll
          for (int mt = 0; mt < S::kTiles; ++mt) {
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint32_t rows[4] = {a[mt][part].x, a[mt][part].y, a[mt][part].z, a[mt][part].w};
              if (dot == 0 && part == 0) mma<true>(score[mt][n], rows, b0, b1);
              else mma<false>(score[mt][n], rows, b0, b1);
            }
          }
        }
      }
    }

    // value scales as 2^(base + exponent) * value
    float value[kSubs], exponent[kSubs], undo[kSubs];
    bool near = true;
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      value[sub] = scales[4 + sub] * unit;
      exponent[sub] = 0.0f;
      undo[sub] = 1.0f;
      near = near && __float_as_uint(scales[4 + sub]) - least < (kScales + 1u) << 23;
    }
    if (!near) {  // (the same for the warp) the first scale, zeros, scales far from the first, infinities
      int field[kSubs], largest = 0;
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        field[sub] = static_cast<int>(__float_as_uint(scales[4 + sub]) >> 23 & 0xffu);
        if (field[sub] < 255) largest = max(largest, field[sub]);
      }
      int base = least == kNoScale ? min(max(largest + 1, kLeastField), 254) : static_cast<int>(least >> 23) + kScales;
      if (largest > base + kMostAbove) {
        const int up = largest - base - kMostAbove, lower = min(up, kMostLower) & ~1, less = up - lower;
        const float by0 = power2(-(less >> 1)), by1 = power2((less >> 1) - less);
        base += up;
#pragma unroll
        for (int at = 0; at < MODE; ++at) {
          sums.m[at] -= lower;
          sums.l[at] *= power2(lower);
#pragma unroll
          for (int j = 0; j < SIZE / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums.o[at][j][i] = sums.o[at][j][i] * by0 * by1;
        }
      }
      far = max(far, largest - base);
      if (largest > 0) least = static_cast<uint32_t>(base - kScales) << 23;
      unit = power2(127 - base + kLift);
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const int e = field[sub] - base;
        value[sub] = scales[4 + sub] * unit;
        if (field[sub] == 0 || field[sub] == 255) {
          value[sub] = field[sub] == 0 ? 0.0f : NAN;
          exponent[sub] = -kZeroBelow;
        } else if (e > 0 || e < -kScales) {
          value[sub] = __uint_as_float((__float_as_uint(scales[4 + sub]) & 0x807fffffu) | (127u + kLift) << 23);
          if (e < -kZeroBelow) value[sub] *= power2(max(e + kZeroBelow, -126));
          exponent[sub] = static_cast<float>(max(e, -kZeroBelow));
        }
        undo[sub] = power2(-static_cast<int>(exponent[sub]));
      }
    }
    // the rows' scores and their maxima
    float x[MODE][2 * kSubs][2], most[MODE];
    bool moves = false;
#pragma unroll
    for (int at = 0; at < MODE; ++at) {
#pragma unroll
      for (int n = 0; n < 2 * kSubs; ++n) {
        const float f = factor[at] * scales[n / 2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float* c = score[at / 2][n];
          x[at][n][i] = fmaf(MODE == kPacked ? c[i] + c[2 + i] : c[at % 2 * 2 + i], f, exponent[n / 2]);
        }
      }
    }
    if (key > common - kKeys) {  // (the same for the warp) columns 2 quad and 2 quad + 1
#pragma unroll
      for (int at = 0; at < MODE; ++at)
#pragma unroll
        for (int n = 0; n < 2 * kSubs; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (key + n * 8 + quad + 4 * i >= limit[at]) x[at][n][i] = -INFINITY;
    }
#pragma unroll
    for (int at = 0; at < MODE; ++at) {
      most[at] = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2 * kSubs; ++n) most[at] = fmaxf(most[at], fmaxf(x[at][n][0], x[at][n][1]));
      most[at] = fmaxf(most[at], __shfl_xor_sync(0xffffffffu, most[at], 1));
      most[at] = fmaxf(most[at], __shfl_xor_sync(0xffffffffu, most[at], 2));
      moves = moves || fabsf(most[at] - sums.m[at]) > kWindow;
    }
    if (__any_sync(0xffffffffu, moves)) {
      const float room = power2(kRoom - far);  // (the weighted values are at most 2^(far + 14) times the weights' sum)
#pragma unroll
      for (int at = 0; at < MODE; ++at) {
        const float old = sums.m[at], next = 2.0f * ceilf(0.5f * most[at]) - kAbove;
        float held = fmaxf(sums.l[at], __shfl_xor_sync(0xffffffffu, sums.l[at], 1));
        held = fmaxf(held, __shfl_xor_sync(0xffffffffu, held, 2));
        const bool falls = most[at] < old - kWindow && most[at] > -INFINITY && held < room;
        const float now = most[at] > old + kWindow ? next : falls ? fmaxf(next, old - kDown) : old;
        const float r = now == old ? 1.0f : power2(max(static_cast<int>(0.5f * (old - now)), -126));
        sums.m[at] = now;
        sums.l[at] *= r * r;
        const float r0 = __shfl_sync(0xffffffffu, r, quad * 8), r1 = __shfl_sync(0xffffffffu, r, quad * 8 + 4);
#pragma unroll
        for (int j = 0; j < SIZE / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sums.o[at][j][i] = sums.o[at][j][i] * (i & 1 ? r1 : r0) * (i & 1 ? r1 : r0);
      }
    }
    uint32_t weight[MODE][kWeights][2 * kSubs];
#pragma unroll
    for (int at = 0; at < MODE; ++at) {
#pragma unroll
      for (int n = 0; n < 2 * kSubs; ++n) {
        const float e0 = exp2_of(x[at][n][0] - sums.m[at]), e1 = exp2_of(x[at][n][1] - sums.m[at]);
        sums.l[at] = fmaf(e0 + e1, undo[n / 2], sums.l[at]);
        uint32_t lo;
        split(e0 * value[n / 2], e1 * value[n / 2], weight[at][0][n], lo);
        if (kWeights == 2) weight[at][kWeights - 1][n] = lo;
      }
    }
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      uint32_t v[4][kValueWords];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // keys of columns 2 quad, 2 quad + 1 of both 8-key tiles
        read_words<kValueWords>(slot + (i & 1 ? value_at ^ 64 : value_at) + (sub * 16 + 4 * i) * SIZE, v[i]);
#pragma unroll
      for (int w = 0; w < kValueWords; ++w) {
        uint32_t b[4][2];  // of the word's four elements: keys 0-7, keys 8-15
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          to_halves<STORAGE>(interleave<STORAGE>(v[2 * pair][w], v[2 * pair + 1][w], 0), b[0][pair], b[1][pair]);
          to_halves<STORAGE>(interleave<STORAGE>(v[2 * pair][w], v[2 * pair + 1][w], 1), b[2][pair], b[3][pair]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t values[4] = {b[2 * i][0], b[2 * i + 1][0], b[2 * i][1], b[2 * i + 1][1]};
#pragma unroll
          for (int at = 0; at < MODE; ++at)
#pragma unroll
            for (int part = 0; part < kWeights; ++part)
              mma<false>(sums.o[at][w * 2 + i], values, weight[at][part][2 * sub], weight[at][part][2 * sub + 1]);
        }
      }
    }
  }
  wait_groups<0>();
  // From units of 2^(base - kLift) to ones, which other warps and blocks have
  // too: most of it moves the reference, what could leave the range of the sum of
  // the weights scales the values.
  const int base = least == kNoScale ? 0 : static_cast<int>(least >> 23) + kScales - 127, fold = max(base - 10, -10);
  const float to_l = power2(-fold), to_o = power2(base - kLift - fold);
#pragma unroll
  for (int at = 0; at < MODE; ++at) {
    sums.m[at] += fold;
    sums.l[at] += __shfl_xor_sync(0xffffffffu, sums.l[at], 1);
    sums.l[at] += __shfl_xor_sync(0xffffffffu, sums.l[at], 2);
    sums.l[at] *= to_l;
#pragma unroll
    for (int j = 0; j < SIZE / 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums.o[at][j][i] *= to_o;
  }
}

// SHARED: of the keys behind those that all sequences have in common, whose sums are joined at the end.
template <int SIZE, int STORAGE, int MODE, int LO, bool SHARED>
__global__ void __launch_bounds__(kThreads, resident_of(MODE)) attention_kernel(const __grid_constant__ Plan p) {
  constexpr int kRows = rows_of(MODE);
  extern __shared__ __align__(128) char shared[];
  __shared__ int scan[kGroups], found[5];
  __shared__ float most[kGroups][kRows], total[kGroups][kRows], factors[kRows];
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  pdl_wait();
  const int pages = SHARED ? common_pages(p.a, p.shared, found) : 0;
  if (SHARED) __syncthreads();  // (found is used again)
  Walk<tile_keys(SIZE)> walk;
  if (!begin_walk<tile_keys(SIZE), kGroups>(p, pages, scan, found, &walk)) return;
  Segment seg;
  while (walk.next(p, &seg)) {
    const int b = seg.b, head = seg.item / p.blocks, first_row = seg.item % p.blocks * kRows;
    if (seg.empty) {
      for (int i = threadIdx.x; i < kRows * SIZE / 4; i += kThreads) {
        const int row = first_row + i / (SIZE / 4);
        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row < p.rows) store4(p, out_row<SIZE>(p, b, head, row) + i % (SIZE / 4) * 4, zero);
      }
      continue;
    }
    Sums<SIZE, MODE> sums;
    const int item = p.a.dtype == CB_F32 ? 4 : 2;
    const void* query = static_cast<const char*>(p.a.q) + static_cast<long long>(b) * p.a.q_strides[0] * item;
    warp_item<SIZE, STORAGE, MODE, LO>(p, query, seg.s, head, first_row, seg.tile, seg.tiles, shared, factors, sums);

    // join the groups
    __syncthreads();  // every warp is done with the ring
    float* rows = reinterpret_cast<float*>(shared);  // (groups, kRows, kPitch)
    constexpr int kPitch = SIZE + 4;                 // (neighbouring rows begin in different banks)
    static_assert(kGroups * kRows * kPitch * 4 <= shared_bytes(SIZE, MODE, LO), "the rows to join fit the ring");
#pragma unroll
    for (int at = 0; at < MODE; ++at) {
      if ((lane & 3) == 0) {
        most[group][at * 8 + (lane >> 2)] = sums.m[at];
        total[group][at * 8 + (lane >> 2)] = sums.l[at];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float* to = rows + (group * kRows + at * 8 + 2 * (lane & 3) + n) * kPitch + element_of<SIZE>(lane >> 2);
#pragma unroll
        for (int j = 0; j < SIZE / 16; j += 2)
          *reinterpret_cast<float4*>(to + 2 * j) =
              make_float4(sums.o[at][j][n], sums.o[at][j][2 + n], sums.o[at][j + 1][n], sums.o[at][j + 1][2 + n]);
      }
    }
    __syncthreads();
    float* partial = part_of<SIZE, kRows>(p, blockIdx.x, seg.begins);
    for (int i = threadIdx.x; i < kRows * SIZE / 4; i += kThreads) {
      const int r = i / (SIZE / 4), d = i % (SIZE / 4) * 4;
      float top = -INFINITY, sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kGroups; ++w) top = fmaxf(top, most[w][r]);
#pragma unroll
      for (int w = 0; w < kGroups; ++w) {
        const float f = most[w][r] == -INFINITY ? 0.0f : root2_of(most[w][r] - top);
        const float4 x = *reinterpret_cast<const float4*>(rows + (w * kRows + r) * kPitch + d);
        sum += f * total[w][r] * f;
        v[0] += f * x.x * f; v[1] += f * x.y * f; v[2] += f * x.z * f; v[3] += f * x.w * f;
      }
      const int row = first_row + r;
      if (seg.whole) {
        if (row < p.rows) {
          if (SHARED && pages > 0 && row / p.group < seg.s.row.count)
            add_shared<SIZE>(p, pages, static_cast<long long>(b) * p.rows + row, head, d, &top, &sum, v);
          const bool real = row / p.group < seg.s.row.count && sum != 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = real ? v[k] / sum : 0.0f;
          store4(p, out_row<SIZE>(p, b, head, row) + d, v);
        }
      } else {
        *reinterpret_cast<float4*>(partial + 2 * kRows + r * SIZE + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) {
          partial[r] = top;
          partial[kRows + r] = sum;
        }
      }
    }
    if (!seg.whole) {
      __syncthreads();
      if (threadIdx.x == 0) found[0] = last_part(p, seg);
      __syncthreads();
      if (found[0])  // (its first part is the first of its block's range, or the second)
        join<SIZE, kRows, SHARED>(p, b, head, first_row, seg.s.row.count, seg.last - seg.from + 1,
                                  part_of<SIZE, kRows>(p, seg.from, seg.from_begins),
                                  part_of<SIZE, kRows>(p, seg.from, true), pages, threadIdx.x, kThreads);
    }
    __syncthreads();  // the joined rows are read; the ring is free again
  }
}

// ---- launch --------------------------------------------------------------------

template <int SIZE, int STORAGE, int MODE, int LO, bool SHARED>
int resident_blocks() {
  static thread_local int device = -1, per_sm = 0;
  int now = 0;
  cudaGetDevice(&now);
  if (now != device) {
    auto kernel = attention_kernel<SIZE, STORAGE, MODE, LO, SHARED>;
    constexpr int kShared = shared_bytes(SIZE, MODE, LO);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, kShared) != cudaSuccess)
      per_sm = 0;
    device = per_sm > 0 ? now : -1;
  }
  return per_sm;
}

// Calls f with the template arguments of a launch: blocks of 8 rows, 16, 24 or
// 32 by the rows of a kv head, of 24 or 32 those that need fewer blocks (16 x
// 5100 keys on average, int8, bfloat16: 8 rows 41 us, 12 and 16 45 and 46; 20
// rows 60 in one block of 24 and 68 in one of 32; 40 rows 102 in two of 24 and
// 118 in two of 32).
template <typename F>
long long with_variant(const cb_paged_attention_args& a, F f) {
  const long long rows = a.tokens * (a.heads / a.cache.kv_heads);
  auto by_rows = [&](auto size, auto storage) {
    const auto two = std::integral_constant<int, 2>{};
    const auto none = std::integral_constant<int, kNoParts>{};
    if (rows <= 8) return f(size, storage, std::integral_constant<int, kPacked>{}, none);
    auto by_type = [&](auto mode) {
      if (a.dtype == CB_F32) return f(size, storage, mode, std::integral_constant<int, kBothParts>{});
      if (a.dtype == CB_F16) return f(size, storage, mode, std::integral_constant<int, kWeightParts>{});
      return f(size, storage, mode, none);
    };
    if (rows <= 16) return by_type(two);
    if ((rows + 23) / 24 == (rows + 31) / 32) return by_type(std::integral_constant<int, 3>{});
    return by_type(std::integral_constant<int, 4>{});
  };
  auto by_storage = [&](auto size) {
    return a.cache.storage == CB_I8 ? by_rows(size, std::integral_constant<int, CB_I8>{})
                                    : by_rows(size, std::integral_constant<int, CB_E4M3>{});
  };
  if (a.cache.head_size == 32) return by_storage(std::integral_constant<int, 32>{});
  if (a.cache.head_size == 64) return by_storage(std::integral_constant<int, 64>{});
  return by_storage(std::integral_constant<int, 128>{});
}

}  // namespace

long long attention_scratch(const cb_paged_attention_args& a, bool shared) {
  if (a.batch == 0 || a.tokens == 0) return 0;
  return with_variant(a, [&](auto size, auto storage, auto mode, auto lo) -> long long {
    const int per_sm = shared ? resident_blocks<size.value, storage.value, mode.value, lo.value, true>()
                              : resident_blocks<size.value, storage.value, mode.value, lo.value, false>();
    return grid_of(a, rows_of(mode.value), tile_keys(size.value), per_sm) * 8LL *
           partial_floats(size.value, rows_of(mode.value));
  });
}

int launch_attention(const cb_paged_attention_args& a, const SharedKeys* shared, void* scratch, unsigned* counters,
                     cudaStream_t stream) {
  const char* who = shared != nullptr ? "cb_paged_attention_shared" : "cb_paged_attention";
  CB_REQUIRE(a.q != nullptr && a.out != nullptr && counters != nullptr, "%s: a null pointer", who);
  CB_REQUIRE(reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && reinterpret_cast<uintptr_t>(scratch) % 16 == 0,
             "%s: out and scratch must be 16-byte aligned", who);
  return static_cast<int>(with_variant(a, [&](auto size, auto storage, auto mode, auto lo) -> long long {
    constexpr int SIZE = size.value, STORAGE = storage.value, MODE = mode.value, LO = lo.value;
    auto go = [&](auto kernel, int per_sm) -> int {
      CB_REQUIRE(per_sm >= 1 && per_sm <= 8, "%s: %d blocks of the kernel fit an SM", who, per_sm);
      const long long grid = grid_of(a, rows_of(MODE), tile_keys(SIZE), per_sm);
      CB_REQUIRE(grid > 0, "%s: %lld rows of up to %lld keys are too many for one call", who,
                 a.batch * a.heads * a.tokens, a.cache.columns * a.cache.page);
      CB_REQUIRE(scratch != nullptr, "%s: a null pointer", who);
      Plan p = plan_of(a, rows_of(MODE), scratch, counters);
      p.shared = shared != nullptr ? *shared : SharedKeys{};
      launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), shared_bytes(SIZE, MODE, LO), stream, true, p);
      return check_launch(who);
    };
    if (shared != nullptr)
      return go(attention_kernel<SIZE, STORAGE, MODE, LO, true>, resident_blocks<SIZE, STORAGE, MODE, LO, true>());
    return go(attention_kernel<SIZE, STORAGE, MODE, LO, false>, resident_blocks<SIZE, STORAGE, MODE, LO, false>());
  }));
}

}  // namespace cb

using namespace cb;

extern "C" {

long long cb_paged_attention_scratch(const cb_paged_attention_args* args) {
  if (args == nullptr || attention_check(*args, "cb_paged_attention") != CB_OK) return 0;
  return attention_scratch(*args, false);
}

long long cb_paged_attention_counters(const cb_paged_attention_args* args) {
  if (args == nullptr || attention_check(*args, "cb_paged_attention") != CB_OK) return 0;
  return 8LL * sm_count();  // more than any launch has blocks
}

int cb_paged_attention(const cb_paged_attention_args* args, void* scratch, unsigned* counters, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_paged_attention: null arguments");
  const int status = attention_check(*args, "cb_paged_attention");
  if (status != CB_OK) return status;
  if (args->batch == 0 || args->tokens == 0) return CB_OK;
  return launch_attention(*args, nullptr, scratch, counters, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
