// Page operations of the paged KV cache: cb_pages_extend, _fork, _truncate,
// _compact, _copy.
//
// The book is whole numbers, and every result is the one that the slots
// handled one after the other in the order of the call would give: ranks are
// prefix sums over the block, and where several slots drop or copy the same
// page the choice goes by position, never by which atomic came first.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Exclusive prefix sum of v in thread order; *total receives the sum.
__device__ __forceinline__ long long block_scan(long long v, long long* shared, long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();  // shared may still be read
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    long long w = shared[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    shared[lane] = w;
  }
  __syncthreads();
  *total = shared[kWarps - 1];
  return incl - v + (warp > 0 ? shared[warp - 1] : 0);
}

// Scratch of cb_pages_extend and cb_pages_compact: the pages to copy (their
// number, sources and targets), then lists of the kernel.
struct Copies {
  int* count;
  int* source;
  int* target;
  int* more;
};
__host__ __device__ __forceinline__ Copies copies_of(void* scratch, long long n) {
  int* p = static_cast<int*>(scratch);
  return {p, p + 4, p + 4 + n, p + 4 + 2 * n};
}

__global__ void __launch_bounds__(kThreads) extend_kernel(cb_page_book k, const int* counts, const int* sequences,
                                                          long long n, void* scratch, int* flag) {
  __shared__ long long shared[kWarps];
  const Copies copies = copies_of(scratch, n);
  int* tails = copies.more;      // open last page of each slot, or -1
  int* plan = copies.more + n;   // pages it takes, negative - 1 where the first of them is a copy
  int* firsts = copies.more + 2 * n;
  if (threadIdx.x == 0) *copies.count = 0;
  bool bad = false;
  for (long long i = threadIdx.x; i < n; i += kThreads) {
    const long long slot = sequences != nullptr ? sequences[i] : i;
    int tail = -1;
    if (slot < 0 || slot >= k.slots || counts[i] < 0) {
      bad = true;
    } else {
      const int length = k.lengths[slot];
      if (length < 0 || length > k.columns * k.page) bad = true;
      else if (length % k.page != 0 && counts[i] > 0) {
        tail = k.table[slot * k.columns + length / k.page];
        if (tail < 0 || tail >= k.pages) bad = true;
      }
      for (long long j = 0; j < i && sequences != nullptr; ++j) bad = bad || sequences[j] == slot;
    }
    tails[i] = tail;
  }
  bool outgrown = false;
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    return;
  }
  long long taken_before = 0, copied_before = 0;
  for (long long at = 0; at < n; at += kThreads) {
    const long long i = at + threadIdx.x;
    int taken = 0;
    bool copied = false;
    if (i < n) {
      const long long slot = sequences != nullptr ? sequences[i] : i;
      const long long length = k.lengths[slot], grown = length + counts[i];
      const long long have = (length + k.page - 1) / k.page, need = (grown + k.page - 1) / k.page;
      outgrown = outgrown || need > k.columns;
      const int tail = tails[i];
      if (tail >= 0 && k.refs[tail] > 1) {
        int earlier = 0;
        for (long long j = 0; j < i; ++j) earlier += tails[j] == tail;
        copied = k.refs[tail] - earlier > 1;
      }
      taken = need > k.columns ? 0 : static_cast<int>(need - have) + (copied ? 1 : 0);
    }
    long long total;
    const long long rank = block_scan((static_cast<long long>(copied) << 32) + taken, shared, &total);
    if (i < n) {
      plan[i] = copied ? -taken - 1 : taken;
      firsts[i] = static_cast<int>(taken_before + (rank & 0xffffffffll));
      if (copied) copies.source[copied_before + (rank >> 32)] = static_cast<int>(i);
    }
    taken_before += total & 0xffffffffll;
    copied_before += total >> 32;
  }
  const int height = *k.height;
  // __syncthreads_or also orders the lists above before their use below
  if (__syncthreads_or(outgrown || taken_before > height || height > k.pages)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_PAGES);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (long long i = threadIdx.x >> 5; i < n; i += kWarps) {
    const long long slot = sequences != nullptr ? sequences[i] : i;
    const bool copied = plan[i] < 0;
    const int taken = copied ? -plan[i] - 1 : plan[i];
    const int base = (k.lengths[slot] + k.page - 1) / k.page - (copied ? 1 : 0);
    for (int m = lane; m < taken; m += 32) {
      const int page = k.free_pages[height - 1 - firsts[i] - m];
      if (page < 0 || page >= k.pages) {
        raise_flag(flag, CB_FLAG_BOOK);
        continue;
      }
      k.table[slot * k.columns + base + m] = page;
      k.refs[page] = 1;
    }
  }
  __syncthreads();
  for (long long r = threadIdx.x; r < copied_before; r += kThreads) {
    const int i = copies.source[r];
    const long long slot = sequences != nullptr ? sequences[i] : i;
    copies.target[r] = k.table[slot * k.columns + k.lengths[slot] / k.page];
    copies.source[r] = tails[i];
    atomicSub(&k.refs[tails[i]], 1);
  }
  __syncthreads();
  for (long long i = threadIdx.x; i < n; i += kThreads)
    k.lengths[sequences != nullptr ? sequences[i] : i] += counts[i];
  if (threadIdx.x == 0) {
    *k.height = height - static_cast<int>(taken_before);
    *copies.count = static_cast<int>(copied_before);
  }
}

__global__ void __launch_bounds__(256) fork_kernel(cb_page_book k, const int* parents, const int* children,
                                                   long long n, int* flag) {
  const long long i = blockIdx.x;
  const int parent = parents[i], child = children[i];
  bool bad = parent < 0 || parent >= k.slots || child < 0 || child >= k.slots;
  for (long long j = threadIdx.x; j < n; j += blockDim.x)
    bad = bad || (j != i && children[j] == child) || parents[j] == child;
  if (!bad) bad = k.lengths[child] != 0 || k.lengths[parent] < 0 || k.lengths[parent] > k.columns * k.page;
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    return;
  }
  const int length = k.lengths[parent];
  for (long long m = threadIdx.x; m < k.columns; m += blockDim.x) {
    const int page = k.table[parent * k.columns + m];
    k.table[child * k.columns + m] = page;
    if (m * k.page < length) {
      if (page >= 0 && page < k.pages) atomicAdd(&k.refs[page], 1);
      else raise_flag(flag, CB_FLAG_BOOK);
    }
  }
  __syncthreads();  // every thread has seen the child empty
  if (threadIdx.x == 0) k.lengths[child] = length;
}

// Entry e = i * columns + m of the call is dropped where need <= m < have of
// slot i.  A page that nobody holds any more is claimed by the last of its
// dropped entries: refs[page] goes from 0 to -(e + 1), the least of them.
__global__ void __launch_bounds__(kThreads) truncate_kernel(cb_page_book k, const int* counts, const int* sequences,
                                                            long long n, int* flag) {
  __shared__ long long shared[kWarps];
  bool bad = false;
  for (long long i = threadIdx.x; i < n; i += kThreads) {
    const long long slot = sequences != nullptr ? sequences[i] : i;
    if (slot < 0 || slot >= k.slots) {
      bad = true;
      continue;
    }
    const int length = k.lengths[slot];
    bad = bad || length < 0 || length > k.columns * k.page || (counts != nullptr && (counts[i] < 0 || counts[i] > length));
    for (long long j = 0; j < i && sequences != nullptr; ++j) bad = bad || sequences[j] == slot;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    return;
  }
  const long long entries = n * k.columns;
  auto dropped = [&](long long e) -> int* {
    const long long i = e / k.columns, m = e % k.columns;
    const long long slot = sequences != nullptr ? sequences[i] : i;
    const long long length = k.lengths[slot], rest = counts != nullptr ? length - counts[i] : 0;
    const bool drop = m * k.page < length && m * k.page >= rest;
    return drop ? k.table + slot * k.columns + m : nullptr;
  };
  for (long long e = threadIdx.x; e < entries; e += kThreads) {
    const int* at = dropped(e);
    if (at == nullptr) continue;
    if (*at >= 0 && *at < k.pages) atomicSub(&k.refs[*at], 1);
    else raise_flag(flag, CB_FLAG_BOOK);
  }
  __syncthreads();
  for (long long e = threadIdx.x; e < entries; e += kThreads) {
    const int* at = dropped(e);
    if (at == nullptr || *at < 0 || *at >= k.pages) continue;
    if (__ldcg(&k.refs[*at]) <= 0) atomicMin(&k.refs[*at], static_cast<int>(-(e + 1)));
  }
  __syncthreads();
  long long pushed = *k.height;
  for (long long done = 0; done < entries; done += kThreads) {
    const long long e = entries - 1 - done - threadIdx.x;
    int* at = e >= 0 ? dropped(e) : nullptr;
    const int page = at != nullptr ? *at : -1;
    const bool mine = page >= 0 && page < k.pages && __ldcg(&k.refs[page]) == static_cast<int>(-(e + 1));
    long long total;
    const long long rank = block_scan(mine ? 1 : 0, shared, &total);
    if (mine) {
      if (pushed + rank < k.pages) k.free_pages[pushed + rank] = page;
      else raise_flag(flag, CB_FLAG_BOOK);
      k.refs[page] = 0;
    }
    if (at != nullptr) *at = -1;
    pushed += total;
  }
  __syncthreads();
  for (long long i = threadIdx.x; i < n; i += kThreads) {
    const long long slot = sequences != nullptr ? sequences[i] : i;
    k.lengths[slot] = counts != nullptr ? k.lengths[slot] - counts[i] : 0;
  }
  if (threadIdx.x == 0) *k.height = static_cast<int>(pushed < k.pages ? pushed : k.pages);
}

__global__ void __launch_bounds__(kThreads) compact_kernel(cb_page_book k, void* scratch, int* flag) {
  __shared__ long long shared[kWarps];
  const Copies copies = copies_of(scratch, k.pages);
  int* to = copies.more;
  long long held = 0;
  for (long long at = 0; at < k.pages; at += kThreads) {
    const long long p = at + threadIdx.x;
    if (p < k.pages) to[p] = static_cast<int>(p);
    held += __syncthreads_count(p < k.pages && k.refs[p] > 0);
  }
  long long holes = 0, moves = 0;
  for (long long at = 0; at < k.pages; at += kThreads) {
    const long long p = at + threadIdx.x;
    const bool live = p < k.pages && k.refs[p] > 0;
    const bool hole = p < held && !live, move = p >= held && live;
    long long total;
    const long long rank = block_scan((static_cast<long long>(move) << 32) + (hole ? 1 : 0), shared, &total);
    if (hole) copies.target[holes + (rank & 0xffffffffll)] = static_cast<int>(p);
    if (move) copies.source[moves + (rank >> 32)] = static_cast<int>(p);
    holes += total & 0xffffffffll;
    moves += total >> 32;
  }
  __syncthreads();
  for (long long r = threadIdx.x; r < moves; r += kThreads) {
    const int source = copies.source[r], target = copies.target[r];
    to[source] = target;
    k.refs[target] = k.refs[source];
    k.refs[source] = 0;
  }
  __syncthreads();
  for (long long e = threadIdx.x; e < k.slots * k.columns; e += kThreads) {
    const int page = k.table[e];
    if (page >= k.pages) raise_flag(flag, CB_FLAG_BOOK);
    else if (page >= held) k.table[e] = to[page];
  }
  for (long long i = threadIdx.x; i < k.pages - held; i += kThreads)
    k.free_pages[i] = static_cast<int>(k.pages - 1 - i);
  if (threadIdx.x == 0) {
    *k.height = static_cast<int>(k.pages - held);
    *copies.count = static_cast<int>(moves);
  }
}

// Copies of whole pages: unit u = (copy, layer, K or V).
__global__ void __launch_bounds__(256) copy_kernel(cb_page_pools p, const int* source, const int* target,
                                                   const int* count, long long n, int* flag) {
  const long long copies = count != nullptr ? *count : n;
  const long long units = copies * p.layers * 2;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long r = u / (p.layers * 2), layer = u / 2 % p.layers;
    const int from = source[r], to = target[r];
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
      if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
      continue;
    }
    char* pool = static_cast<char*>(u % 2 ? p.v_pages : p.k_pages) + layer * p.pages * p.page_bytes;
    float* scale = (u % 2 ? p.v_scale : p.k_scale) + layer * p.pages * p.kv_heads;
    const uint4* src = reinterpret_cast<const uint4*>(pool + from * p.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(pool + to * p.page_bytes);
    for (long long i = threadIdx.x; i < p.page_bytes / 16; i += blockDim.x) dst[i] = src[i];
    for (int i = threadIdx.x; i < p.kv_heads; i += blockDim.x)
      scale[static_cast<long long>(to) * p.kv_heads + i] = scale[static_cast<long long>(from) * p.kv_heads + i];
  }
}

int book_check(const cb_page_book* k, long long n, const char* who) {
  CB_REQUIRE(k != nullptr && k->table && k->lengths && k->refs && k->free_pages && k->height, "%s: a null pointer", who);
  CB_REQUIRE(k->slots >= 1 && k->columns >= 1 && k->pages >= 1 && k->page >= 1, "%s: an empty book", who);
  CB_REQUIRE(k->pages < (1LL << 31) && k->columns * k->page < (1LL << 31) && k->slots * k->columns < (1LL << 31),
             "%s: %lld slots of %lld columns, %lld pages", who, k->slots, k->columns, k->pages);
  CB_REQUIRE(n >= 0 && n <= k->slots, "%s: %lld of %lld slots", who, n, k->slots);
  return CB_OK;
}

int pools_check(const cb_page_pools* p, const char* who) {
  CB_REQUIRE(p != nullptr && p->k_pages && p->v_pages && p->k_scale && p->v_scale, "%s: a null pointer", who);
  CB_REQUIRE(p->layers >= 1 && p->pages >= 1 && p->kv_heads >= 1 && p->page_bytes > 0 && p->page_bytes % 16 == 0,
             "%s: %lld layers of %lld pages of %lld bytes", who, p->layers, p->pages, p->page_bytes);
  CB_REQUIRE(reinterpret_cast<uintptr_t>(p->k_pages) % 16 == 0 && reinterpret_cast<uintptr_t>(p->v_pages) % 16 == 0,
             "%s: the pools must be 16-byte aligned", who);
  return CB_OK;
}

int launch_copies(const cb_page_pools& p, const int* source, const int* target, const int* count, long long most,
                  int* flag, cudaStream_t stream) {
  const long long units = most * p.layers * 2, cap = 8LL * sm_count();
  copy_kernel<<<static_cast<unsigned>(units < cap ? units : cap), 256, 0, stream>>>(p, source, target, count, most,
                                                                                  flag);
  return check_launch("cb_pages: copies");
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_pages_scratch(const cb_page_book* book, long long n) {
  // extend: five lists of n; compact: three of the pages
  const long long extend = 5 * n, compact = 3 * book->pages;
  return 4 * (4 + (extend > compact ? extend : compact));
}

int cb_pages_extend(const cb_page_book* book, const cb_page_pools* pools, const int* counts, const int* sequences,
                    long long n, void* scratch, int* error_flag, cb_stream_t stream) {
  int status = book_check(book, n, "cb_pages_extend");
  if (status == CB_OK) status = pools_check(pools, "cb_pages_extend");
  if (status != CB_OK) return status;
  if (n == 0) return CB_OK;
  CB_REQUIRE(counts != nullptr && scratch != nullptr, "cb_pages_extend: a null pointer");
  CB_REQUIRE(pools->pages == book->pages, "cb_pages_extend: %lld pages in the pools, %lld in the book", pools->pages,
             book->pages);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  extend_kernel<<<1, kThreads, 0, s>>>(*book, counts, sequences, n, scratch, error_flag);
  status = check_launch("cb_pages_extend");
  if (status != CB_OK) return status;
  const Copies c = copies_of(scratch, n);
  return launch_copies(*pools, c.source, c.target, c.count, n, error_flag, s);
}

int cb_pages_fork(const cb_page_book* book, const int* parents, const int* children, long long n, int* error_flag,
                  cb_stream_t stream) {
  const int status = book_check(book, n, "cb_pages_fork");
  if (status != CB_OK) return status;
  if (n == 0) return CB_OK;
  CB_REQUIRE(parents != nullptr && children != nullptr, "cb_pages_fork: a null pointer");
  fork_kernel<<<static_cast<unsigned>(n), 256, 0, static_cast<cudaStream_t>(stream)>>>(*book, parents, children, n,
                                                                                     error_flag);
  return check_launch("cb_pages_fork");
}

int cb_pages_truncate(const cb_page_book* book, const int* counts, const int* sequences, long long n, int* error_flag,
                      cb_stream_t stream) {
  const int status = book_check(book, n, "cb_pages_truncate");
  if (status != CB_OK) return status;
  if (n == 0) return CB_OK;
  truncate_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(*book, counts, sequences, n, error_flag);
  return check_launch("cb_pages_truncate");
}

int cb_pages_compact(const cb_page_book* book, const cb_page_pools* pools, void* scratch, int* error_flag,
                     cb_stream_t stream) {
  int status = book_check(book, 0, "cb_pages_compact");
  if (status == CB_OK) status = pools_check(pools, "cb_pages_compact");
  if (status != CB_OK) return status;
  CB_REQUIRE(scratch != nullptr, "cb_pages_compact: a null pointer");
  CB_REQUIRE(pools->pages == book->pages, "cb_pages_compact: %lld pages in the pools, %lld in the book", pools->pages,
             book->pages);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  compact_kernel<<<1, kThreads, 0, s>>>(*book, scratch, error_flag);
  status = check_launch("cb_pages_compact");
  if (status != CB_OK) return status;
  const Copies c = copies_of(scratch, book->pages);
  return launch_copies(*pools, c.source, c.target, c.count, book->pages, error_flag, s);
}

int cb_pages_copy(const cb_page_pools* pools, const int* source, const int* target, long long n, int* error_flag,
                  cb_stream_t stream) {
  const int status = pools_check(pools, "cb_pages_copy");
  if (status != CB_OK) return status;
  CB_REQUIRE(n >= 0, "cb_pages_copy: %lld pages", n);
  if (n == 0) return CB_OK;
  CB_REQUIRE(source != nullptr && target != nullptr, "cb_pages_copy: a null pointer");
  return launch_copies(*pools, source, target, nullptr, n, error_flag, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
