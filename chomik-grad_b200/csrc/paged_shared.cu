// Attention over the paged 8-bit KV cache for sequences that begin alike:
// cb_paged_attention_shared.
//
// The result is cb_paged_attention's.  Sequences that were forked from one hold
// the same pages from their beginning on; what they all hold is read and
// multiplied once, with the rows of all sequences together, and each
// sequence's own keys by cb_paged_attention's kernel, which joins both.
//
// For row r (a sequence's query, one of a kv head's group) and the keys j of P, the
// common pages, and T, the sequence's own:
//   y_j = scale log2(e) ks_j (q_r . kq_j) + log2 vs_j
//   O = sum_j 2^(y_j - c) vq_j,  l = sum_j 2^(y_j - c) / vs_j    over P, and over T
//   out = (2^(c_P - m) O_P + 2^(c_T - m) O_T) / (2^(c_P - m) l_P + 2^(c_T - m) l_T)
// Whether a value scale is part of the weight or of the values is a matter of
// notation, so O needs no scaled copy of the codes.
//
// What bounds it: with R rows to a key the products are 2 R flops a byte (64 samples
// of 4 rows to a kv head, or 16 blocks of 20: 256 and 320 rows), so they go to
// tcgen05: 128-row products of fp16 (codes are exact in it) with float32 sums in
// tensor memory.  A tile of 64 keys of 128 elements then takes a set of 128 rows 640
// cycles on the tensor cores (scores 8 x 48, values 4 x 64), but 8192 exponentials with their
// conversions about 1700 cycles on the four schedulers: that, and the hand-offs
// between warps that it delays, is what is left (2600 to 2900 cycles a tile of two
// sets, 3400 where the weights have two parts; 64 samples of 16384 keys 83 us on the
// device, 91 in float16 and 95 in float32, 16 blocks of 5 tokens at 32700 keys 154 and
// 177 in float16, by cb_paged_attention, each sequence for itself, 351 and 292; 8
// samples of 32768 keys, both sets the same rows, 65 and 72).
//
// Three launches, each begun while the one before ends: the common pages of each
// sequence; the shared keys, a block to an SM, whose warps are divided by what they
// do (two sets of 128 rows share a tile of keys and values, 20 warps); the tails.
#include <type_traits>

#include "paged_attention.cuh"
#include "tc_core.cuh"

namespace cb {
namespace {

constexpr int kCommonThreads = 128;

// For each sequence of the call: the whole pages that its table row has in
// common with that of the first sequence that takes part, no more than leave a
// key of its own to each row.
__global__ void __launch_bounds__(kCommonThreads) common_kernel(const cb_paged_attention_args a, int* common) {
  __shared__ int reference, differs;
  const int b = blockIdx.x, thread = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (thread == 0) reference = differs = INT_MAX;
  __syncthreads();
  PagedRow row;
  for (int first = 0; first < a.batch && reference == INT_MAX; first += kCommonThreads) {
    const bool there = first + thread < a.batch && paged_row(a.cache, a.sequences, a.counts, a.tokens, first + thread,
                                                             a.error_flag, &row) && row.count > 0;
    __syncthreads();  // (everyone has looked at `reference`)
    if (there) atomicMin(&reference, first + thread);
    __syncthreads();
  }
  const bool takes_part = paged_row(a.cache, a.sequences, a.counts, a.tokens, b, a.error_flag, &row) && row.count > 0;
  if (!takes_part) {  // (the same for the block)
    if (thread == 0) {
      common[b] = INT_MAX;
      if (b == 0) common[a.batch] = reference == INT_MAX ? 0 : a.sequences != nullptr ? a.sequences[reference] : reference;
    }
    return;
  }
  const int slot = a.sequences != nullptr ? a.sequences[reference] : reference;
  const int* other = a.cache.table + slot * a.cache.columns;
  const int limit = (row.length - row.count) / a.cache.page;
  constexpr int kEach = 4;
  for (int first = 0; first < limit && differs == INT_MAX; first += kEach * kCommonThreads) {
    int mine = INT_MAX;
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i) {
      const int at = first + i * kCommonThreads + thread;
      if (at < limit && row.table[at] != other[at]) mine = at;
    }
    __syncthreads();  // (everyone has looked at `differs`)
    if (mine != INT_MAX) atomicMin(&differs, mine);
    __syncthreads();
  }
  if (thread == 0) {
    common[b] = min(limit, differs);
    if (b == 0) common[a.batch] = slot;
  }
}

struct SharedPlan {
  cb_paged_attention_args a;
  int group, rows;  // query heads of a kv head; rows of a kv head in a sequence
  bool wide;        // queries can be read 16 bytes at a time
  SharedKeys shared;
  float* parts;
};

// ---- the shared keys -------------------------------------------------------------

constexpr int kRowLanes = 128;  // rows of a product: lanes of the tensor memory
constexpr int kSetThreads = 128;
// Warps 0 and 1 issue the products of the two sets of rows, 2 looks up pages and scales:
// first, since a scheduler prefers its older warps, and these wait most and do least.
constexpr int kIssueWarp = 0, kLookWarp = 2, kWeighWarp = 4, kKeyWarp = 12, kValueWarp = 16;
constexpr int kSharedThreads = 32 * (kValueWarp + 4);
// Registers of a thread, 96 at the launch: of the warps that weigh, of those that
// convert, and of the four that issue and look up (61440 of a block, before and after;
// the launch checks that they were there before, since a raise waits for them).
constexpr int kWeighRegisters = 152, kConvertRegisters = 72, kIssueRegisters = 32;
constexpr int kBlockRegisters =
    32 * (8 * kWeighRegisters + 8 * kConvertRegisters + 4 * kIssueRegisters);
constexpr int kStages = 3, kAhead = 3;  // tiles as fp16, and tiles whose codes are on their way
constexpr int kChunkBytes = kSharedTile * 128;  // 64 keys of 64 fp16 elements
// Columns of the tensor memory: weighted values of both sets; then, for each set, the
// scores of a tile and behind them its weights as fp16: of two tiles by turns, or high
// and low parts of one, 16 keys of each together.
constexpr int kValuesAt = 0, kScoresAt = 256, kSetColumns = 128, kWeightsAt = 64, kColumns = 512;
__host__ __device__ constexpr int weights_at(bool lo, int tile) { return kWeightsAt + (lo ? 0 : (tile & 1) * 32); }

// Of a tile's four runs of 16 keys: the line of each in the pools (page and kv head; -1:
// none), and its scales, of values as log2, 2^-log2 and what the logarithm leaves.
// They are looked up for eight tiles at a time, a lane to a run.
constexpr int kBatch = 8, kBatches = 3;
// Warps that read a batch, and arrive when they have left it: those that weigh and those
// that convert.  (Neither follows from the other: with one set of rows, whose tiles are
// weighed by turns, the values may be converted eight tiles behind the scores.)
constexpr int kBatchReaders = kValueWarp + 4 - kWeighWarp;
struct __align__(16) Runs {
  long long line[4];
  float key[4], log[4], inverse[4], factor[4];
  int irregular, pad[3];
};

template <int SIZE>
struct SharedShape {
  static constexpr int kChunks = SIZE == 128 ? 2 : 1;
  static constexpr int kStageBytes = 2 * kChunks * kChunkBytes;  // keys, then values
  static constexpr int kCodeBytes = 2 * kSharedTile * SIZE;      // of a tile on its way
  static constexpr int kQueryBytes = kChunks * kRowLanes * 128;  // of a set, or of one part
  // (the tiles begin on 1024)
  static constexpr int kBytes = kStages * kStageBytes + 2 * kQueryBytes + kAhead * kCodeBytes + 1024;
  static constexpr int kWide = SIZE < 64 ? 64 : SIZE;            // columns of the weighted values
};
// Every block asks for the shared memory of the largest, so that no other that takes
// tensor memory fits beside it: it takes all of that before the kernels ahead have ended,
// and one of theirs, or of those behind, that waited for some on the same SM would keep both.
constexpr int kBlockBytes = SharedShape<128>::kBytes;
static_assert(kBlockBytes >= SharedShape<64>::kBytes && kBlockBytes >= SharedShape<32>::kBytes, "the largest");

// What has a second fp16 part, of what the first leaves: nothing (bfloat16), the weights
// (float16, whose queries are exact in one), queries and weights (float32).  One part of
// the weights would do for 11-bit outputs but for an error as large as their rounding:
// 2.9e-4 of the result against 2.1e-4 (152 us against 176 for 16 blocks of 5 tokens at
// 32700 keys, 81 against 90 for 64 samples of 16384).
enum { kOnePart = 0, kWeightParts = 1, kBothParts = 2 };
__host__ __device__ constexpr bool low_queries(int parts) { return parts == kBothParts; }
__host__ __device__ constexpr bool low_weights(int parts) { return parts != kOnePart; }

// fp16 x fp16 -> float32, 128 x n; the second operand with its contraction along (K) or across its rows.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool across) {
  return (1u << 4) | (across ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (128u >> 4 << 24);
}
// A tile of rows of 128 bytes whose contraction runs across them: 64 columns to a
// chunk, chunks kChunkBytes apart, 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t across_desc(const void* tile) {
  return ((static_cast<uint64_t>(smem_addr(tile)) >> 4) & 0x3FFFull) |
         (static_cast<uint64_t>(kChunkBytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void multiply(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// The same with its first operand in shared memory.
__device__ __forceinline__ void multiply_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void store8(uint32_t at, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Every lane of the warp waits for a phase and looks at most kPolls
// times, without the clock, a read of which takes longer than most of these waits.
// QUICK: by mbarrier.test_wait, which does not suspend the thread; a try_wait that
// began well before its phase ends returns about a thousand cycles after it.
constexpr uint32_t kPolls = 1u << 24;
template <bool QUICK = true>
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  bool there = true;
  for (uint32_t i = 0;; ++i) {
    if (QUICK) {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(smem_addr(bar)), "r"(parity)
          : "memory");
      if (done != 0) break;
    } else if (mbar_try_wait_short(bar, parity)) {
      break;
    }
    if (i == kPolls || ((i & 255u) == 255u && *abort != 0)) {
      there = false;
      break;
    }
  }
  return __all_sync(0xffffffffu, there);
}
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void unpack_row8(const SharedPlan& p, const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = *reinterpret_cast<const __half2*>(w + i);
    const bool brain = p.a.dtype == CB_BF16;
    x[2 * i] = brain ? __uint_as_float(w[i] << 16) : __low2float(h);
    x[2 * i + 1] = brain ? __uint_as_float(w[i] & 0xffff0000u) : __high2float(h);
  }
}
// Eight neighbouring elements of a query row: float32 (WIDE), or of 16 bits.
template <bool WIDE>
__device__ __forceinline__ void load_row8(const SharedPlan& p, long long at, float* x) {
  if (WIDE) {
    const float* from = static_cast<const float*>(p.a.q) + at;
    if (p.wide) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(from + i);
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = from[i];
    }
  } else {
    const uint16_t* from = static_cast<const uint16_t*>(p.a.q) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = from[2 * i] | static_cast<uint32_t>(from[2 * i + 1]) << 16;
    unpack_row8(p, make_uint4(w[0], w[1], w[2], w[3]), x);
  }
}
// 32 float32 columns of this thread's lane of the tensor memory (warp-wide).
// The load and the wait for it are one statement: between two, the compiler could
// move registers that are not written yet.
__device__ __forceinline__ void load32(uint32_t at, float* out) {
  uint32_t v[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
      "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) out[i] = __uint_as_float(v[i]);
}

// What the roles of a block walk: `count` tiles from tile `first` of each of its items.
struct SharedWalk {
  int blocks, keys, item, step, items, first, tiles, count;  // step: to the block's next item; count: of all its tiles
  SharedCut cut;
  const int* table;
};

// Barriers of a block.  Sets and stages count their phases apart.
struct SharedSync {
  uint64_t key_full[kStages], key_free[kStages], value_full[kStages], value_free[kStages];
  uint64_t batch_full[kBatches], batch_free[kBatches], query_full, query_free, all_done;
  uint64_t score_full[2], score_free[2];
  uint64_t weight_full[2][2], value_done[2][2];  // [set][tile % 2]: a set is up to two tiles ahead of its products
  uint32_t tmem;
  int abort, found[2];
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// Looks up the runs of the range's tiles.  (Through L2: the kernels ahead may have written
// the table and the scales after this one began, so they are no read-only data of it.)
__device__ __forceinline__ bool look_up(const SharedPlan& p, const SharedWalk& w, Runs* runs, SharedSync& sync) {
  const cb_paged_cache& c = p.a.cache;
  const int lane = threadIdx.x & 31, run = lane & 3, count = w.count, shift = 31 - __clz(c.page);
#pragma unroll 1
  for (int batch = 0; batch * kBatch < count; ++batch) {
    const int n = batch * kBatch + lane / 4, key = (w.first + n % w.tiles) * kSharedTile + run * 16;
    const int head = (w.item + n / w.tiles * w.step) / w.blocks, slot = batch % kBatches;
    long long line = -1;
    if (n < count && key < w.keys) {
      const int page = __ldcg(w.table + (key >> shift));
      if (static_cast<unsigned>(page) < static_cast<unsigned>(c.pages)) line = static_cast<long long>(page) * c.kv_heads + head;
      else raise_flag(p.a.error_flag, CB_FLAG_BOOK);
    }
    const bool real = line >= 0;
    const float k = real ? __ldcg(c.k_scale + line) : 0.0f, v = real ? __ldcg(c.v_scale + line) : 1.0f;
    float log = -INFINITY, inverse = 0.0f, factor = 1.0f;
    if (real) {  // (an error of the logarithm moves the weights and their sum alike)
      const float size = fabsf(v);
      log = isfinite(v) ? fmaxf(__log2f(size), -100.0f) : 0.0f;
      inverse = exp2_of(-log);
      factor = !isfinite(v) ? NAN : size < 7.9e-31f ? v * 1.2676506002282294e30f : v < 0.0f ? -1.0f : 1.0f;  // 2^-100, 2^100
    }
    const unsigned regular = __ballot_sync(0xffffffffu, v >= 9.3e-10f && v <= 1.07e9f && k >= 0.0f);  // 2^-30 .. 2^30
    if (batch >= kBatches && !wait_warp<false>(sync.batch_free + slot, static_cast<uint32_t>((batch / kBatches - 1) & 1), &sync.abort))
      return false;
    Runs& to = runs[slot * kBatch + lane / 4];
    to.line[run] = line;
    to.key[run] = k;
    to.log[run] = log;
    to.inverse[run] = inverse;
    to.factor[run] = factor;
    if (run == 0) to.irregular = (regular >> lane & 15u) != 15u;
    mbar_arrive(sync.batch_full + slot);
  }
  return true;
}

// Keys (or values) of the range's tiles: codes to fp16 in shared memory, rows of 64
// elements on 128 bytes, their 16-byte pieces exchanged as the products read them.  The
// codes of the next kAhead tiles are copied to shared memory meanwhile; a thread
// converts what it copied, so nothing but its own copies has to be waited for.  One
// copy of this code serves both: what the roles run by turns has to fit the
// instruction cache (with 80 KB of unrolled code a tile took 5900 cycles).
template <int SIZE, int STORAGE>
__device__ __forceinline__ bool convert(const SharedPlan& p, const SharedWalk& w, bool values, char* tiles, char* codes,
                                        const Runs* runs, SharedSync& sync) {
  constexpr int kPieces = SIZE / 16, kLoads = kSharedTile * kPieces / kSetThreads, kRows = kSetThreads / kPieces;
  const cb_paged_cache& c = p.a.cache;
  const int thread = threadIdx.x % kSetThreads, piece = thread % kPieces, row = thread / kPieces;
  const int count = w.count;
  const char* pool = static_cast<const char*>(values ? c.v_pages : c.k_pages) + piece * 16;
  const uint32_t codes_at = smem_addr(codes) + thread * 16;
  if (values && SIZE == 32) {  // the columns that no element has
    for (int i = thread; i < kStages * kSharedTile * 4; i += kSetThreads)
      *reinterpret_cast<uint4*>(tiles + i / (kSharedTile * 4) * SharedShape<SIZE>::kStageBytes +
                                tc::swizzle_offset(i / 4 % kSharedTile, 4 + i % 4)) = make_uint4(0, 0, 0, 0);
  }
  uint64_t* const free = values ? sync.value_free : sync.key_free;
  uint64_t* const full = values ? sync.value_full : sync.key_full;
  bool ok = true;
  int stage = 0, turn = 0, slot = 0;
  int next = 0, next_tile = 0, batch = 0, batch_turn = 0;  // what is copied next
#pragma unroll 1
  for (int n = -kAhead; n < count; ++n) {
    if (n >= 0) {
      if (turn > 0 && ok) ok = wait_warp<false>(free + stage, static_cast<uint32_t>((turn - 1) & 1), &sync.abort);
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      const int first = piece % 4 * 2;
      const bool turned = piece >= 4;  // (so that both chunks' pieces of a row touch different banks)
      char* to = tiles + stage * SharedShape<SIZE>::kStageBytes + piece / 4 * kChunkBytes;
      const char* from = codes + slot * SharedShape<SIZE>::kCodeBytes + thread * 16;
      uint2 v[kLoads], u[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        v[i] = *reinterpret_cast<const uint2*>(from + i * kSetThreads * 16 + 8 * turned);
        u[i] = *reinterpret_cast<const uint2*>(from + i * kSetThreads * 16 + 8 * !turned);
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = row + i * kRows;
        uint4 h;
        to_halves<STORAGE>(v[i].x, h.x, h.y);
        to_halves<STORAGE>(v[i].y, h.z, h.w);
        *reinterpret_cast<uint4*>(to + tc::swizzle_offset(r, first + turned)) = h;
        to_halves<STORAGE>(u[i].x, h.x, h.y);
        to_halves<STORAGE>(u[i].y, h.z, h.w);
        *reinterpret_cast<uint4*>(to + tc::swizzle_offset(r, first + !turned)) = h;
      }
      tc::fence_async_shared();
      mbar_arrive(full + stage);
      if (++stage == kStages) {
        stage = 0;
        ++turn;
      }
    }
    if (next < count) {
      if (next % kBatch == 0 && ok) ok = wait_warp<false>(sync.batch_full + batch, static_cast<uint32_t>(batch_turn & 1), &sync.abort);
      const Runs& tile = runs[batch * kBatch + next % kBatch];
      long long line[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) line[i] = tile.line[(row + i * kRows) / 16];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int in = ((w.first + next_tile) * kSharedTile + row + i * kRows) & (c.page - 1);
        const bool real = ok && line[i] >= 0;
        copy16(codes_at + slot * SharedShape<SIZE>::kCodeBytes + i * kSetThreads * 16,
               pool + (real ? (line[i] * c.page + in) * SIZE : 0), real);
      }
      ++next;
      if (++next_tile == w.tiles) next_tile = 0;
      if (next % kBatch == 0) {
        __syncwarp();  // (every lane has its lines of the batch, which may be looked up anew from here on)
        if ((threadIdx.x & 31) == 0) mbar_arrive(sync.batch_free + batch);
        if (++batch == kBatches) {
          batch = 0;
          ++batch_turn;
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++slot == kAhead) slot = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  return ok;
}

// Issues the products of a set over the block's range: a warp, so that what it computes
// is uniform, and one lane of it.  Both sets take every tile (SETS 2: their own rows)
// or every other one (1: the same rows).  A tile's scores are computed as soon as those
// of the one before are in registers, while the set weighs it.  (While warps take
// exponentials, a look at a barrier can wait for hundreds of cycles: those for the
// tiles come before the one for the weights.)
template <int SIZE, int SETS, int PARTS>
__device__ __forceinline__ bool issue(const SharedWalk& w, int set, const char* keys, const char* values,
                                      const char* queries, SharedSync& sync) {
  using S = SharedShape<SIZE>;
  constexpr uint32_t kScoreDesc = idesc_f16(kSharedTile, false), kValueDesc = idesc_f16(S::kWide, true);
  volatile int* abort = &sync.abort;
  const uint32_t tmem = __shfl_sync(0xffffffffu, sync.tmem, 0);
  const bool leads = elected();
  const uint64_t query = tc::sw128_desc(queries + (SETS == 2 ? set * S::kQueryBytes : 0));
  int iteration = 0, segment = 0, before = 0;  // tiles of the set; tiles before the segment
#pragma unroll 1
  for (int item = w.item; item < w.items; item += w.step, ++segment) {
    const int jobs = SETS == 2 ? w.tiles : (w.tiles - set + 1) / 2;
    if (!wait_warp(&sync.query_full, static_cast<uint32_t>(segment & 1), abort)) return false;
    tc::fence_after();
#pragma unroll 1
    for (int job = -1; job < jobs; ++job) {
      if (job + 1 < jobs) {  // the scores of the next tile
        const int n = before + (SETS == 2 ? job + 1 : 2 * (job + 1) + set), now = iteration + job + 1;
        if (!wait_warp(sync.key_full + n % kStages, static_cast<uint32_t>(n / kStages & 1), abort) ||
            (now > 0 && !wait_warp(sync.score_free + set, static_cast<uint32_t>((now - 1) & 1), abort)))
          return false;
        tc::fence_after();
        const uint64_t tile = tc::sw128_desc(keys + n % kStages * S::kStageBytes);
        const uint32_t d = tmem + kScoresAt + set * kSetColumns;
        if (leads) {
#pragma unroll
          for (int part = 0; part < (low_queries(PARTS) ? 2 : 1); ++part)
#pragma unroll
            for (int k = 0; k < SIZE / 16; ++k)
              multiply_shared(d, query + (part * S::kQueryBytes + k / 4 * kRowLanes * 128 + k % 4 * 32) / 16,
                              tile + (k / 4 * kChunkBytes + k % 4 * 32) / 16, kScoreDesc, part + k > 0);
          tc::umma_commit(sync.score_full + set);
          tc::umma_commit(sync.key_free + n % kStages);
        }
        __syncwarp();
      }
      if (job >= 0) {  // the weighted values of tile `job`
        const int n = before + (SETS == 2 ? job : 2 * job + set), now = iteration + job, buffer = now & 1;
        if (!wait_warp(sync.value_full + n % kStages, static_cast<uint32_t>(n / kStages & 1), abort) ||
            !wait_warp(sync.weight_full[set] + buffer, static_cast<uint32_t>(now / 2 & 1), abort))
          return false;
        tc::fence_after();
        const uint64_t tile = across_desc(values + n % kStages * S::kStageBytes);
        const uint32_t d = tmem + kValuesAt + set * 128, a = tmem + kScoresAt + set * kSetColumns + weights_at(low_weights(PARTS), now);
        if (leads) {
#pragma unroll
          for (int part = 0; part < (low_weights(PARTS) ? 2 : 1); ++part)
#pragma unroll
            for (int k = 0; k < kSharedTile / 16; ++k)
              multiply(d, a + k * (low_weights(PARTS) ? 16 : 8) + part * 8, tile + k * 2048 / 16, kValueDesc, job > 0 || part + k > 0);
          tc::umma_commit(sync.value_done[set] + buffer);
          tc::umma_commit(sync.value_free + n % kStages);
        }
        __syncwarp();
      }
    }
    if (leads) tc::umma_commit(&sync.query_free);
    __syncwarp();
    iteration += jobs;
    before += w.tiles;
  }
  return true;
}

// The references follow the scores and value scales (their logarithms included) as
// in paged_attention.cuh: what multiplies the value codes is 2^(y - c), y a key's
// score plus the logarithm of its value scale.  A tile whose largest is more
// than kRise above c or `fall` below it moves c to kRest below it: it is rounded to
// 2^-24 of 2^(y - c), so the largest of every tile keeps 11 bits, and those 2^5 below it;
// of two parts it keeps 16 (float16) and 22 (float32, which falls earlier).  Moving takes a pass over the sums (2000 cycles); the range
// makes it rare (rises of 15 and falls of 6: most tiles of some row, 137 us for 64
// samples of 16384 keys; falls of 8 or 15: the same 82 us).
// It falls as far as the sums against it stay below 2^kHeldExponent: keys below about
// 2^-100 of all the weights before them may be lost.
constexpr float kRise = 15.0f, kRest = 2.0f, kFarBelow = 60.0f;
constexpr int kHeldExponent = 100, kLargeExponent = 112;
__host__ __device__ constexpr float fall_of(bool close) { return close ? 2.0f : 8.0f; }
// e of 2^e <= x < 2^(e + 1); -127 of zero, 128 of infinity and NaN
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }

// Two float32 numbers in a 64-bit register, for the instructions that take both.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void split_pair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// x = 2^(x * by + shift) of 16 numbers, and their sum.  Half of them for 16-bit
// outputs are computed on the multiply-add units (the special function unit would take
// 512 cycles for a warp's tile, and two warps share it): 2^e = 2^n 2^f with n the
// nearest whole number to e (added to 1.5 * 2^23, whose low bits it becomes), and 2^f,
// |f| <= 1/2, by its Taylor polynomial of degree 5: (f ln 2)^6 / 720 < 2.5e-6, a
// hundredth of the weights' rounding to 11 bits.  (2^n is multiplied: added to the
// exponent's bits it would make a number of a NaN.)
template <bool CLOSE>
__device__ __forceinline__ float exponentials(float* x, float by, float shift) {
  const uint64_t by2 = pair_of(by, by), shift2 = pair_of(shift, shift);
  uint64_t run[2] = {0, 0};
  constexpr float kMagic = 12582912.0f, kLn2 = 0.6931471805599453f;
  const uint64_t magic = pair_of(kMagic, kMagic), back = pair_of(-kMagic, -kMagic), minus = pair_of(-1.0f, -1.0f);
#pragma unroll
  for (int k = 0; k < 16; k += 2) {
    uint64_t e = fma2(pair_of(x[k], x[k + 1]), by2, shift2);
    float a, b;
    split_pair(e, a, b);
    if (CLOSE || k % 4 == 0) {
      x[k] = exp2_of(a);
      x[k + 1] = exp2_of(b);
    } else {
      asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(a));  // -126
      asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(b));
      e = pair_of(a, b);
      const uint64_t n = add2(e, magic), f = fma2(add2(n, back), minus, e);
      constexpr float c1 = kLn2, c2 = kLn2 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4, c5 = c4 * kLn2 / 5;
      uint64_t y = fma2(pair_of(c5, c5), f, pair_of(c4, c4));
      y = fma2(y, f, pair_of(c3, c3));
      y = fma2(y, f, pair_of(c2, c2));
      y = fma2(y, f, pair_of(c1, c1));
      y = fma2(y, f, pair_of(1.0f, 1.0f));
      split_pair(n, a, b);
      const uint64_t power = pair_of(__uint_as_float((__float_as_uint(a) << 23) + 0x3f800000u),
                                     __uint_as_float((__float_as_uint(b) << 23) + 0x3f800000u));
      split_pair(mul2(y, power), x[k], x[k + 1]);
    }
    run[k / 2 & 1] = add2(run[k / 2 & 1], pair_of(x[k], x[k + 1]));
  }
  float a, b;
  split_pair(add2(run[0], run[1]), a, b);
  return a + b;
}

// 2^a, also where it is below the least normal number: a row's sum of weights is
// against a reference that holds the value scale, up to 2^127, and keeps what is far
// below its largest.
__device__ __forceinline__ float weight_of(float a) {
  return a < 0.0f ? exp2_of(a + 64.0f) * 5.421010862427522e-20f : exp2_of(a);  // 2^-64
}

// Sixteen weights as fp16, and what is left of them.
template <bool LO>
__device__ __forceinline__ void store_weights(uint32_t at, const float* x) {
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
    hi[k] = bits(h);
    if (LO) lo[k] = bits(__floats2half2_rn(x[2 * k] - __low2float(h), x[2 * k + 1] - __high2float(h)));
  }
  store8(at, hi);
  if (LO) store8(at + 8, lo);
}

// A set of 128 rows, a thread each.
template <int SIZE, int STORAGE, int SETS, int PARTS>
__device__ __forceinline__ bool weigh(const SharedPlan& p, const SharedWalk& w, char* queries, float* factors, long long* offsets,
                                      const Runs* runs, SharedSync& sync) {
  const int thread = threadIdx.x - 32 * kWeighWarp, set = thread / kSetThreads, r = thread % kSetThreads;
  const int local = SETS == 2 ? thread : r;
  volatile int* abort = &sync.abort;
  const uint32_t lanes = sync.tmem + (static_cast<uint32_t>(r / 32 * 32) << 16);
  const uint32_t sums = lanes + kValuesAt + set * 128, scores = lanes + kScoresAt + set * kSetColumns;
  const int all_rows = static_cast<int>(p.a.batch) * p.rows;
  // every warp takes every batch of runs and leaves it, whether it weighs a tile of it or not
  int batch = -1;
  auto reach = [&](int n) {  // the batch of the range's tile n
    while (batch < n / kBatch) {
      __syncwarp();
      if (batch >= 0 && (threadIdx.x & 31) == 0) mbar_arrive(sync.batch_free + batch % kBatches);
      ++batch;
      if (!wait_warp(sync.batch_full + batch % kBatches, static_cast<uint32_t>(batch / kBatches & 1), abort)) return false;
    }
    return true;
  };
  int iteration = 0, segment = 0, before = 0;
#pragma unroll 1
  for (int item = w.item; item < w.items; item += w.step, ++segment) {
    const int tiles = w.tiles, head = item / w.blocks;
    const int row = item % w.blocks * p.shared.block_rows + local;
    const bool real = row < all_rows, any = __any_sync(0xffffffffu, real);  // (rows of no warp are skipped)

    // the warp's rows of queries, SIZE / 8 lanes to a row, scaled to below 2, in the
    // order of the codes' halves
    long long from = -1;
    if (real) {
      const int b = row / p.rows, t = row % p.rows / p.group, h = head * p.group + row % p.group;
      from = b * p.a.q_strides[0] + t * p.a.q_strides[1] + h * p.a.q_strides[2];
    }
    offsets[thread] = from;
    __syncwarp();
    if (segment > 0 && !wait_warp(&sync.query_free, static_cast<uint32_t>((segment - 1) & 1), abort)) return false;
    const uint32_t turn_of_queries = static_cast<uint32_t>(segment & 1);
    if (SETS == 2 || low_queries(PARTS) || set == 0) {
      // 16-bit rows are copied to where they will be first; the loops are rolled, since
      // code that runs once costs its way to the instruction cache
      constexpr int kLanes = SIZE / 8;
      const int lane = threadIdx.x & 31, d = lane % kLanes * 8;
      char* to = queries + (SETS == 2 || low_queries(PARTS) ? set * SharedShape<SIZE>::kQueryBytes : 0) + d / 64 * kRowLanes * 128;
      const bool copied = !low_queries(PARTS) && p.wide;
      if (copied) {
#pragma unroll 1
        for (int step = 0; step < kLanes; ++step) {
          const int from_lane = step * (32 / kLanes) + lane / kLanes;
          const long long at_row = offsets[thread / 32 * 32 + from_lane];
          copy16(smem_addr(to + tc::swizzle_offset(r / 32 * 32 + from_lane, d % 64 / 8)),
                 static_cast<const uint16_t*>(p.a.q) + (at_row >= 0 ? at_row + d : 0), at_row >= 0);
        }
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      }
#pragma unroll 1
      for (int step = 0; step < kLanes; ++step) {
        const int from_lane = step * (32 / kLanes) + lane / kLanes, local_row = r / 32 * 32 + from_lane;
        const long long at_row = offsets[thread / 32 * 32 + from_lane];
        uint4* place = reinterpret_cast<uint4*>(to + tc::swizzle_offset(local_row, d % 64 / 8));
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, largest = 0.0f;
        if (copied) unpack_row8(p, *place, x);
        else if (at_row >= 0) load_row8<low_queries(PARTS)>(p, at_row + d, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        const int e = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -126), 127);
        const float down = e == 127 ? 5.877471754111438e-39f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        const float sign = p.a.scale < 0.0f ? -down : down;
        if (d == 0) factors[set * kSetThreads + local_row] = fabsf(p.a.scale) * 1.4426950408889634f * power2(e);
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int first = STORAGE == CB_I8 ? i / 2 * 4 + i % 2 : 2 * i, second = STORAGE == CB_I8 ? first + 2 : first + 1;
          const float a = x[first] * sign, b = x[second] * sign;
          const __half2 hi = __floats2half2_rn(a, b);
          h[i] = low_queries(PARTS) && set == 1 ? bits(__floats2half2_rn(a - __low2float(hi), b - __high2float(hi))) : bits(hi);
        }
        *place = make_uint4(h[0], h[1], h[2], h[3]);
      }
      tc::fence_async_shared();
    }
    mbar_arrive(&sync.query_full);
    __syncwarp();
    // (one part of one set of rows: the other set has its factors from there)
    const bool other = SETS == 1 && !low_queries(PARTS) && set == 1;
    if (other && !wait_warp(&sync.query_full, turn_of_queries, abort)) return false;
    const float factor = factors[other ? r : thread];

    float c = 0.0f, l = 0.0f, sum = 0.0f;  // reference, sum of the weights, and of what multiplied the codes
    float ceiling = 0.0f;                  // a tile whose largest is above it moves c
    bool first = true;
    for (int tile = SETS == 2 ? 0 : set; tile < tiles; tile += SETS == 2 ? 1 : 2, ++iteration) {
      const int n = before + tile;
      const int buffer = iteration & 1;
      const uint32_t weights = scores + weights_at(low_weights(PARTS), iteration);
      if (!reach(n) ||
          !wait_warp(sync.score_full + set, static_cast<uint32_t>(iteration & 1), abort))
        return false;
      tc::fence_after();
      auto leave_scores = [&] {  // they are read: the next tile's may take their place
        tc::fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(sync.score_free + set);
      };
      if (!any) leave_scores();
      if (any) {
        float s[kSharedTile], by[4], log[4], inverse[4];
        const Runs& tile_runs = runs[batch % kBatches * kBatch + n % kBatch];
        const bool irregular = tile_runs.irregular != 0;
        float top = -INFINITY;
        if (__builtin_expect(!irregular, 1)) {
          load32(scores, s);
          load32(scores + 32, s + 32);
          leave_scores();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            by[i] = factor * tile_runs.key[i];
            log[i] = tile_runs.log[i];
            inverse[i] = tile_runs.inverse[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float most = s[16 * i];
#pragma unroll
            for (int k = 1; k < 16; ++k) most = fmaxf(most, s[16 * i + k]);
            top = fmaxf(top, fmaf(most, by[i], log[i]));
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            float x[16];
            tc::tmem_load16(scores + i * 16, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) top = fmaxf(top, fmaf(x[k], factor * tile_runs.key[i], tile_runs.log[i]));
          }
        }
        float now = c;
        if (__any_sync(0xffffffffu, first || top > ceiling || top < c - fall_of(low_queries(PARTS)))) {
          const float next = floorf(top) - kRest;
          if (first) now = top > -INFINITY ? next : 0.0f;
          else if (top > ceiling) now = next;
          else if (top < c - fall_of(low_queries(PARTS)) && top > -INFINITY)  // (the sums stay below 2^kHeldExponent)
            now = fmaxf(next, c - static_cast<float>(max(kHeldExponent - 1 - exponent_of(fmaxf(sum, l)), 0)));
        }
        if (__any_sync(0xffffffffu, first || now != c)) {
          if (!first) {
            // (in two steps: the sum of the weights may be large while c falls by more than 126)
            const float first_step = rintf(0.5f * (c - now)), by0 = exp2_of(first_step), by1 = exp2_of(c - now - first_step);
            l = l * by0 * by1;
            sum = sum * by0 * by1;
            if (!wait_warp(sync.value_done[set] + (buffer ^ 1), static_cast<uint32_t>((iteration - 1) / 2 & 1), abort))
              return false;
            tc::fence_after();
#pragma unroll 1
            for (int d = 0; d < SharedShape<SIZE>::kWide; d += 32) {
              float o[32];
              load32(sums + d, o);
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint32_t v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(o[i + k] * by0 * by1);
                store8(sums + d + i, v);
              }
            }
          }
          c = now;
          ceiling = c + kRise;
        }
        first = false;
        // (low parts leave no room for the weights of two tiles)
        if (low_weights(PARTS) && iteration > 0 &&
            !wait_warp(sync.value_done[set] + (buffer ^ 1), static_cast<uint32_t>((iteration - 1) / 2 & 1), abort))
          return false;
        if (__builtin_expect(!irregular, 1)) {
          // all of a row's far below c: its weights by themselves, since 2^(y - c) may not
          // be there (of that row alone: no bit of a row depends on the rows beside it)
          const bool far = top < c - kFarBelow;
          if (__builtin_expect(__any_sync(0xffffffffu, far), 0)) {
#pragma unroll
            for (int k = 0; k < kSharedTile; ++k)
              l += far && inverse[k / 16] != 0.0f ? weight_of(fmaf(s[k], by[k / 16], -c)) : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float all = exponentials<low_queries(PARTS)>(s + 16 * i, by[i], log[i] - c);
            if (!far) l = fmaf(all, inverse[i], l);
            sum += all;
            store_weights<low_weights(PARTS)>(weights + i * (low_weights(PARTS) ? 16 : 8), s + 16 * i);
          }
        } else {  // value scales of any sign and size: the weights by themselves
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            const float by_i = factor * tile_runs.key[i], shift = tile_runs.log[i] - c, kept = tile_runs.factor[i];
            float x[16], all = 0.0f;
            tc::tmem_load16(scores + i * 16, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float score = x[k] * by_i;
              all += weight_of(score - c);
              x[k] = exp2_of(score + shift);
              sum += x[k];
              x[k] *= kept;
            }
            if (tile_runs.inverse[i] != 0.0f) l += all;
            store_weights<low_weights(PARTS)>(weights + i * (low_weights(PARTS) ? 16 : 8), x);
          }
          // (the weights by themselves are against 2^c over the value scale: up to 2^115 for a key
          // whose values are zero or tiny.  What comes to more lets no tile stay above c.)
          if (exponent_of(l) >= kLargeExponent) ceiling = c + kRest;
          leave_scores();
        }
        tc::tmem_wait_st();
      }
      tc::fence_before();
      mbar_arrive(sync.weight_full[set] + buffer);
    }
    // the part of this set
    const bool some = SETS == 2 || tiles > set;
    if (some && !wait_warp(sync.value_done[set] + ((iteration - 1) & 1), static_cast<uint32_t>((iteration - 1) / 2 & 1), abort))
      return false;
    tc::fence_after();
    if (any) {
      const int rows = p.shared.block_rows;
      const long long piece = static_cast<long long>(item) * w.cut.splits + w.first / w.cut.per;
      float* part = p.parts + (piece * p.shared.ways + (SETS == 2 ? 0 : set)) * rows * (SIZE + 2);
      if (real) {
        part[local] = some ? c : -INFINITY;
        part[rows + local] = l;
      }
#pragma unroll 1
      for (int d = 0; d < SIZE; d += 32) {
        float o[32];
        if (some) {
          load32(sums + d, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        }
        if (real) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float* to = part + 2 * rows + shared_at(rows, local, d + i);
            constexpr int b = STORAGE == CB_I8 ? 2 : 1, e = STORAGE == CB_I8 ? 1 : 2;  // (the order of the codes' halves)
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(o[i]), "f"(o[i + b]),
                         "f"(o[i + e]), "f"(o[i + 3]), "f"(o[i + 4]), "f"(o[i + 4 + b]), "f"(o[i + 4 + e]), "f"(o[i + 7])
                         : "memory");
          }
        }
      }
      tc::fence_before();
    }
    before += tiles;
    if (before < w.count && !reach(before)) return false;
  }
  return true;
}

template <int SIZE, int STORAGE, int SETS, int PARTS>
__global__ void __launch_bounds__(kSharedThreads, 1) shared_kernel(const __grid_constant__ SharedPlan p) {
  using S = SharedShape<SIZE>;
  extern __shared__ char memory[];
  __shared__ SharedSync sync;
  __shared__ Runs runs[kBatches * kBatch];
  __shared__ float factors[2 * kSetThreads];  // what turns a row's products into scores in base 2
  __shared__ long long offsets[2 * kSetThreads];  // of the rows' queries, -1: none
  char* tiles = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(memory) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  // (all of the tensor memory, before the kernels ahead have ended: see kBlockBytes)
  if (warp == kIssueWarp) tc::tmem_alloc(&sync.tmem, kColumns);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(sync.key_full + i, kSetThreads);
      mbar_init(sync.value_full + i, kSetThreads);
      mbar_init(sync.key_free + i, SETS);
      mbar_init(sync.value_free + i, SETS);
    }
    for (int i = 0; i < kBatches; ++i) {
      mbar_init(sync.batch_full + i, 32);
      mbar_init(sync.batch_free + i, kBatchReaders);
    }
    mbar_init(&sync.query_full, 2 * kSetThreads);
    mbar_init(&sync.query_free, 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(sync.score_full + i, 1);
      mbar_init(sync.score_free + i, kSetThreads / 32);
      for (int k = 0; k < 2; ++k) {
        mbar_init(sync.weight_full[i] + k, kSetThreads);
        mbar_init(sync.value_done[i] + k, 1);
      }
    }
    mbar_init(&sync.all_done, 2);
    mbar_fence_init();
    sync.abort = 0;
  }
  tc::fence_before();
  pdl_wait();
  const int pages = common_pages(p.a, p.shared, sync.found);  // (barriers of the block)
  tc::fence_after();
  SharedWalk w;
  w.blocks = static_cast<int>((p.a.batch * p.rows + p.shared.block_rows - 1) / p.shared.block_rows);
  w.keys = pages * p.a.cache.page;
  const int all = p.a.cache.kv_heads * w.blocks, block = static_cast<int>(blockIdx.x);
  w.cut = shared_cut(p.shared, all, w.keys);
  w.item = block / w.cut.splits;
  w.step = w.cut.splits > 1 ? all : static_cast<int>(gridDim.x);
  w.first = block % w.cut.splits * w.cut.per;
  w.tiles = min(w.cut.per, w.cut.tiles - w.first);
  w.items = w.keys > 0 ? all : 0;
  w.count = w.item < w.items ? ((w.items - 1 - w.item) / w.step + 1) * w.tiles : 0;
  w.table = p.a.cache.table + __ldcg(p.shared.common + p.a.batch) * p.a.cache.columns;
  const char* values = tiles + S::kChunks * kChunkBytes;
  char* queries = tiles + kStages * S::kStageBytes;
  char* codes = queries + 2 * S::kQueryBytes;
  bool ok = true;
  if (w.count > 0) {
    if (warp < kWeighWarp) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegisters));
      if (warp < kIssueWarp + 2) ok = issue<SIZE, SETS, PARTS>(w, warp - kIssueWarp, tiles, values, queries, sync);
      if (warp == kLookWarp) ok = look_up(p, w, runs, sync);
    } else if (warp < kKeyWarp) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWeighRegisters));
      ok = weigh<SIZE, STORAGE, SETS, PARTS>(p, w, queries, factors, offsets, runs, sync);
    } else {
      const bool is_value = warp >= kValueWarp;
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegisters));
      ok = convert<SIZE, STORAGE>(p, w, is_value, is_value ? tiles + S::kChunks * kChunkBytes : tiles,
                                  is_value ? codes + S::kCodeBytes / 2 : codes, runs, sync);
    }
    if (!ok) {
      raise_flag(p.a.error_flag, CB_FLAG_WAIT_DATA);
      sync.abort = 1;
    }
  }
  __syncwarp();
  // (arrives once every product that was issued has completed; the lanes that issued them)
  if ((warp == kIssueWarp || warp == kIssueWarp + 1) && elected()) tc::umma_commit(&sync.all_done);
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    // the tensor memory is freed only after the products that write it have completed
    if (!tc::wait_short(&sync.all_done, 0u) && lane == 0) raise_flag(p.a.error_flag, CB_FLAG_WAIT_DRAIN);
    tc::fence_after();
    tc::tmem_dealloc(sync.tmem, kColumns);
  }
}

// Where the pieces of the scratch lie.
struct SharedScratch {
  long long common, attention, parts, bytes;
};
SharedScratch scratch_of(const cb_paged_attention_args& a, const SharedKeys& shared) {
  const long long blocks = (a.batch * a.tokens * (a.heads / a.cache.kv_heads) + shared.block_rows - 1) / shared.block_rows;
  SharedScratch s;
  s.common = 0;
  s.attention = ((a.batch + 1) * 4 + 31) / 32 * 32;
  s.parts = s.attention + (attention_scratch(a, true) + 31) / 32 * 32;
  const long long items = a.cache.kv_heads * blocks, pieces = items > shared.blocks ? items : shared.blocks;
  s.bytes = s.parts + pieces * shared.ways * shared.block_rows * (a.cache.head_size + 2) * 4LL;
  return s;
}
// More than 128 rows of 16-bit queries: two sets of them to a block, which share
// the tiles; float32, whose queries and weights take two parts, and fewer rows: both
// sets are the same rows, and take the tiles in turn.
bool two_sets(const cb_paged_attention_args& a) {
  return a.dtype != CB_F32 && a.batch * a.tokens * (a.heads / a.cache.kv_heads) > kRowLanes;
}
SharedKeys shared_of(const cb_paged_attention_args& a, long long least_bytes) {
  const bool two = two_sets(a);
  SharedKeys s = {};
  s.block_rows = two ? 2 * kRowLanes : kRowLanes;
  s.ways = two ? 1 : 2;
  s.blocks = sm_count();
  s.least = 4;
  s.least_bytes = least_bytes;
  return s;
}

int shared_check(const cb_paged_attention_args& a) {
  const int status = attention_check(a, "cb_paged_attention_shared");
  if (status != CB_OK) return status;
  const long long rows = a.batch * a.tokens * (a.heads / a.cache.kv_heads);
  const long long tiles = (a.cache.columns * a.cache.page + kSharedTile - 1) / kSharedTile;
  const double units = static_cast<double>((rows + kRowLanes - 1) / kRowLanes) * a.cache.kv_heads * tiles;
  CB_REQUIRE(units + (1 << 20) < 2147483648.0 && a.cache.columns * a.cache.page < (1LL << 31) - 4096 && rows < (1LL << 31) - 2 * kRowLanes,
             "cb_paged_attention_shared: %lld rows of up to %lld keys are too many for one call", rows,
             a.cache.columns * a.cache.page);
  return CB_OK;
}

// Whether the sequences could hold enough keys in common for these to be computed apart.
bool may_share(const cb_paged_attention_args& a, const SharedKeys& shared) {
  return worth_sharing(a, shared, a.batch, a.cache.columns * a.cache.page);
}

template <typename F>
int with_shape(const cb_paged_attention_args& a, F f) {
  auto by_rows = [&](auto size, auto storage) {
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    if (a.dtype == CB_F32) return f(size, storage, one, std::integral_constant<int, kBothParts>{});
    auto by_type = [&](auto sets) {
      if (a.dtype == CB_F16) return f(size, storage, sets, std::integral_constant<int, kWeightParts>{});
      return f(size, storage, sets, std::integral_constant<int, kOnePart>{});
    };
    return two_sets(a) ? by_type(two) : by_type(one);
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
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_paged_attention_shared_scratch(const cb_paged_attention_args* args, long long least_bytes) {
  if (args == nullptr || shared_check(*args) != CB_OK || args->batch == 0 || args->tokens == 0) return 0;
  const SharedKeys shared = shared_of(*args, least_bytes);
  return may_share(*args, shared) ? scratch_of(*args, shared).bytes : attention_scratch(*args, false);
}

int cb_paged_attention_shared(const cb_paged_attention_args* args, long long least_bytes, void* scratch,
                              unsigned* counters, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_paged_attention_shared: null arguments");
  const cb_paged_attention_args& a = *args;
  const int status = shared_check(a);
  if (status != CB_OK) return status;
  if (a.batch == 0 || a.tokens == 0) return CB_OK;
  const SharedKeys shared = shared_of(a, least_bytes);
  if (!may_share(a, shared)) return launch_attention(a, nullptr, scratch, counters, static_cast<cudaStream_t>(stream));
  CB_REQUIRE(a.q != nullptr && a.out != nullptr && counters != nullptr && scratch != nullptr,
             "cb_paged_attention_shared: a null pointer");
  CB_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 32 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0,
             "cb_paged_attention_shared: out must be 16-byte aligned, scratch 32");
  // (what launch_attention would refuse, before anything is launched)
  CB_REQUIRE(attention_scratch(a, true) > 0, "cb_paged_attention_shared: %lld rows of up to %lld keys are too many for one call",
             a.batch * a.heads * a.tokens, a.cache.columns * a.cache.page);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  SharedPlan p = {};
  p.a = a;
  p.group = static_cast<int>(a.heads / a.cache.kv_heads);
  p.rows = static_cast<int>(a.tokens * p.group);
  p.shared = shared;
  const SharedScratch at = scratch_of(a, p.shared);
  char* base = static_cast<char*>(scratch);
  int* common = reinterpret_cast<int*>(base + at.common);
  p.shared.common = common;
  p.parts = reinterpret_cast<float*>(base + at.parts);
  p.shared.parts = p.parts;
  const int item = a.dtype == CB_F32 ? 4 : 2;
  p.wide = reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
  for (int i = 0; i < 3; ++i) p.wide = p.wide && a.q_strides[i] * item % 16 == 0;
  const int done = with_shape(a, [&](auto size, auto storage, auto sets, auto parts) -> int {
    constexpr int SIZE = size.value;
    auto kernel = shared_kernel<SIZE, storage.value, sets.value, parts.value>;
    static thread_local int device = -1;
    int now = 0;
    cudaGetDevice(&now);
    if (now != device) {
      cudaFuncAttributes attributes;
      cudaError_t e = cudaFuncGetAttributes(&attributes, kernel);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBlockBytes);
      CB_REQUIRE(e == cudaSuccess, "cb_paged_attention_shared: %s", cudaGetErrorString(e));
      CB_REQUIRE(attributes.numRegs * kSharedThreads >= kBlockRegisters,
                 "cb_paged_attention_shared: built with %d registers a thread, too few to be divided", attributes.numRegs);
      device = now;
    }
    launch(common_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(kCommonThreads), 0, s, true, a, common);
    const int found = check_launch("cb_paged_attention_shared");
    if (found != CB_OK) return found;
    launch(kernel, dim3(static_cast<unsigned>(p.shared.blocks)), dim3(kSharedThreads), kBlockBytes, s, true, p);
    return check_launch("cb_paged_attention_shared");
  });
  if (done != CB_OK) return done;
  return launch_attention(a, &p.shared, base + at.attention, counters, s);
}

}  // extern "C"
