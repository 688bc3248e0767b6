// Attention over the paged 8-bit KV cache for sequences that begin alike:
// cb_paged_attention_shared.
//
// The result is cb_paged_attention's.  Sequences that were forked from one hold
// the same pages from their beginning on; what they all hold is read and
// multiplied once, with the rows of all sequences together, and each
// sequence's own keys by cb_paged_attention's kernel, which joins both.
#include <type_traits>

#include "paged_attention.cuh"

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
  SharedKeys shared;
  float* parts;
};

constexpr int kSimpleThreads = 256;

// A warp to a row.
template <int SIZE>
__global__ void __launch_bounds__(kSimpleThreads) shared_kernel(const __grid_constant__ SharedPlan p) {
  __shared__ int found;
  constexpr int kEach = SIZE / 32;
  const cb_paged_cache& c = p.a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int pages = common_pages(p.shared, p.a.batch, &found);
  if (pages == 0) return;
  const long long all_rows = p.a.batch * p.rows;
  const int blocks = static_cast<int>((all_rows + p.shared.block_rows - 1) / p.shared.block_rows);
  const int items = c.kv_heads * blocks, keys = pages * c.page;
  const SharedCut cut = shared_cut(p.shared, items, keys);
  const int* table = c.table + __ldcg(p.shared.common + p.a.batch) * c.columns;
  const int range = blockIdx.x, end = min((range + 1) * cut.per, items * cut.tiles);
  for (int at = range * cut.per; at < end;) {
    const int item = at / cut.tiles, tile = at % cut.tiles, tiles = min(cut.tiles - tile, end - at);
    const int head = item / blocks;
    float* part = p.parts + static_cast<long long>(item + range) * p.shared.ways * p.shared.block_rows * (SIZE + 2);
    for (int r = warp; r < p.shared.block_rows; r += kSimpleThreads / 32) {
      const long long row = static_cast<long long>(item % blocks) * p.shared.block_rows + r;
      if (row >= all_rows) break;
      const long long b = row / p.rows, t = row % p.rows / p.group, h = head * p.group + row % p.group;
      const long long from = b * p.a.q_strides[0] + t * p.a.q_strides[1] + h * p.a.q_strides[2];
      float q[kEach], o[kEach], m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        q[i] = load_as_f32(p.a.q, from + lane + 32 * i, p.a.dtype);
        o[i] = 0.0f;
      }
      for (int key = tile * kSharedTile; key < min(keys, (tile + tiles) * kSharedTile); ++key) {
        const int page = table[key / c.page];
        if (page < 0 || page >= c.pages) {
          raise_flag(p.a.error_flag, CB_FLAG_BOOK);
          continue;
        }
        const long long at_page = static_cast<long long>(page) * c.kv_heads + head;
        const long long line = (at_page * c.page + key % c.page) * SIZE;
        float dot = 0.0f, v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          float k;
          if (c.storage == CB_I8) {
            k = static_cast<const int8_t*>(c.k_pages)[line + lane + 32 * i];
            v[i] = static_cast<const int8_t*>(c.v_pages)[line + lane + 32 * i];
          } else {
            k = static_cast<float>(static_cast<const __nv_fp8_e4m3*>(c.k_pages)[line + lane + 32 * i]);
            v[i] = static_cast<float>(static_cast<const __nv_fp8_e4m3*>(c.v_pages)[line + lane + 32 * i]);
          }
          dot = fmaf(q[i], k, dot);
        }
        const float x = warp_sum(dot) * (c.k_scale[at_page] * (p.a.scale * 1.4426950408889634f));
        const float now = fmaxf(m, x), keep = exp2f(m - now), w = exp2f(x - now), scaled = w * c.v_scale[at_page];
        l = fmaf(l, keep, w);
#pragma unroll
        for (int i = 0; i < kEach; ++i) o[i] = fmaf(o[i], keep, scaled * v[i]);
        m = now;
      }
      if (lane == 0) {
        part[r] = m;
        part[p.shared.block_rows + r] = l;
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) part[2 * p.shared.block_rows + r * SIZE + lane + 32 * i] = o[i];
    }
    at += tiles;
  }
}

constexpr int kBlockRows = 128;

// Where the pieces of the scratch lie.
struct SharedScratch {
  long long common, attention, parts, bytes;
};
SharedScratch scratch_of(const cb_paged_attention_args& a, const SharedKeys& shared) {
  const long long blocks = (a.batch * a.tokens * (a.heads / a.cache.kv_heads) + shared.block_rows - 1) / shared.block_rows;
  SharedScratch s;
  s.common = 0;
  s.attention = ((a.batch + 1) * 4 + 15) / 16 * 16;
  s.parts = s.attention + (attention_scratch(a, true) + 15) / 16 * 16;
  s.bytes = s.parts + (a.cache.kv_heads * blocks + shared.ranges - 1) * shared.ways * shared.block_rows *
                          (a.cache.head_size + 2) * 4LL;
  return s;
}
SharedKeys shared_of(const cb_paged_attention_args& a) {
  SharedKeys s = {};
  s.block_rows = kBlockRows;
  s.ways = 1;
  s.ranges = sm_count();
  s.least = 1;
  return s;
}

int shared_check(const cb_paged_attention_args& a) {
  const int status = attention_check(a, "cb_paged_attention_shared");
  if (status != CB_OK) return status;
  const long long rows = a.batch * a.tokens * (a.heads / a.cache.kv_heads);
  const long long tiles = (a.cache.columns * a.cache.page + kSharedTile - 1) / kSharedTile;
  const double units = static_cast<double>((rows + kBlockRows - 1) / kBlockRows) * a.cache.kv_heads * tiles;
  CB_REQUIRE(units + (1 << 20) < 2147483648.0,
             "cb_paged_attention_shared: %lld rows of up to %lld keys are too many for one call", rows,
             a.cache.columns * a.cache.page);
  return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_paged_attention_shared_scratch(const cb_paged_attention_args* args) {
  if (args == nullptr || shared_check(*args) != CB_OK || args->batch == 0 || args->tokens == 0) return 0;
  return scratch_of(*args, shared_of(*args)).bytes;
}

int cb_paged_attention_shared(const cb_paged_attention_args* args, void* scratch, unsigned* counters,
                              cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_paged_attention_shared: null arguments");
  const cb_paged_attention_args& a = *args;
  const int status = shared_check(a);
  if (status != CB_OK) return status;
  if (a.batch == 0 || a.tokens == 0) return CB_OK;
  CB_REQUIRE(a.q != nullptr && a.out != nullptr && counters != nullptr && scratch != nullptr,
             "cb_paged_attention_shared: a null pointer");
  CB_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0,
             "cb_paged_attention_shared: out and scratch must be 16-byte aligned");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  SharedPlan p = {};
  p.a = a;
  p.group = static_cast<int>(a.heads / a.cache.kv_heads);
  p.rows = static_cast<int>(a.tokens * p.group);
  p.shared = shared_of(a);
  const SharedScratch at = scratch_of(a, p.shared);
  char* base = static_cast<char*>(scratch);
  int* common = reinterpret_cast<int*>(base + at.common);
  p.shared.common = common;
  p.parts = reinterpret_cast<float*>(base + at.parts);
  p.shared.parts = p.parts;
  launch(common_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(kCommonThreads), 0, s, true, a, common);
  int done = check_launch("cb_paged_attention_shared");
  if (done != CB_OK) return done;
  auto go = [&](auto kernel) {
    launch(kernel, dim3(static_cast<unsigned>(p.shared.ranges)), dim3(kSimpleThreads), 0, s, true, p);
    return check_launch("cb_paged_attention_shared");
  };
  done = a.cache.head_size == 32 ? go(shared_kernel<32>) : a.cache.head_size == 64 ? go(shared_kernel<64>)
                                                                                    : go(shared_kernel<128>);
  if (done != CB_OK) return done;
  return launch_attention(a, &p.shared, base + at.attention, counters, s);
}

}  // extern "C"
