// Page operations of the paged KV cache: cb_pages_extend, _fork, _truncate,
// _compact, _copy.
//
// The book is whole numbers, and every result is the one that the slots
// handled one after the other in the order of the call would give: ranks are
// prefix sums over the block, and where several slots drop or copy the same
// page the choice goes by position, never by which atomic came first.
//
// What bounds them: the book operations read and write some KB to MB in chains
// of dependent steps, so their time is latency; truncate and compact, whose
// lists grow with the table and the pool, run as one cluster of up to eight
// blocks that exchange their counts through distributed shared memory (64
// slots of 128 pages, half of them released: 13 us; by one block 19).  That the
// slots of a call differ is found by comparing all pairs, n^2 / 1024 of them a
// thread.  The copies are bound by memory: a warp for a page of a layer, 8 loads
// of 16 bytes in flight for each lane, a grid that fills the GPU, launched along
// with the book's kernel (programmatic dependent launch), which leaves it the
// list (32 sequences compacted, 16 layers, 1.07 GB read and written: 186 us, of
// which the copies 163 at 6.1 TB/s).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMostBlocks = 8;  // of a cluster: the portable limit
constexpr long long kClusterCopy = 1LL << 20;  // bytes of pages

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

// The sum of `v` (one value of each block) over the blocks before this one, and
// over the cluster.  `slots` is a shared array that no earlier call of the
// kernel used; every thread calls it, and it orders the cluster's memory.
__device__ __forceinline__ long long cluster_scan(long long v, long long* slots, long long* total) {
  cg::cluster_group group = cg::this_cluster();
  const int blocks = static_cast<int>(group.num_blocks()), rank = static_cast<int>(group.block_rank());
  if (static_cast<int>(threadIdx.x) < blocks) *group.map_shared_rank(slots + rank, threadIdx.x) = v;
  cluster_sync();
  long long before = 0, all = 0;
  for (int r = 0; r < blocks; ++r) {
    if (r == rank) before = all;
    all += slots[r];
  }
  *total = all;
  return before;
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

// Copies of whole pages: unit u = (copy, layer, K or V), taken in turn by the
// callers' `warps`, each with kBatch 16-byte loads of a lane in flight.
constexpr int kCopyThreads = 256;
constexpr int kBatch = 8;

__device__ __forceinline__ void copy_units(const cb_page_pools& p, const int* source, const int* target, int copies,
                                           int warp, int warps, int* flag) {
  const unsigned layers = static_cast<unsigned>(p.layers), lane = threadIdx.x & 31;
  const int vectors = static_cast<int>(p.page_bytes / 16);
  const unsigned long long units = 2ull * copies * layers;
  for (unsigned long long u = warp; u < units; u += warps) {
    const unsigned r = static_cast<unsigned>(u / (2 * layers)), rest = static_cast<unsigned>(u % (2 * layers));
    const int from = __ldcg(source + r), to = __ldcg(target + r);
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
      if (lane == 0) raise_flag(flag, CB_FLAG_BOOK);
      continue;
    }
    const long long layer = rest >> 1;
    const bool is_v = rest & 1;
    char* pool = static_cast<char*>(is_v ? p.v_pages : p.k_pages) + layer * p.pages * p.page_bytes;
    float* scale = (is_v ? p.v_scale : p.k_scale) + layer * p.pages * p.kv_heads;
    const uint4* src = reinterpret_cast<const uint4*>(pool + from * p.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(pool + to * p.page_bytes);
    for (int at = lane; at < vectors; at += kBatch * 32) {
      uint4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (at + i * 32 < vectors) v[i] = __ldcs(src + at + i * 32);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (at + i * 32 < vectors) __stcs(dst + at + i * 32, v[i]);
    }
    for (int h = lane; h < p.kv_heads; h += 32)
      scale[static_cast<long long>(to) * p.kv_heads + h] = scale[static_cast<long long>(from) * p.kv_heads + h];
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ cb_page_pools p, const int* source,
                                                            const int* target, const int* count, int n, int* flag) {
  pdl_wait();
  copy_units(p, source, target, count != nullptr ? *count : n, (blockIdx.x * kCopyThreads + threadIdx.x) / 32,
             gridDim.x * (kCopyThreads / 32), flag);
}

__device__ __forceinline__ void extend_book(const cb_page_book& k, const int* counts, const int* sequences,
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
  const int height = *k.height;
  bad = bad || height < 0 || height > k.pages;
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
  // __syncthreads_or also orders the lists above before their use below
  if (__syncthreads_or(outgrown || taken_before > height)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_PAGES);
    return;
  }
  // the pages to take have to be free ones of the pool, each on the stack once:
  // each is marked, before anything else changes
  const int lane = threadIdx.x & 31;
  for (long long r = threadIdx.x; r < taken_before; r += kThreads) {
    const int page = k.free_pages[height - 1 - r];
    bad = bad || page < 0 || page >= k.pages || atomicCAS(&k.refs[page], 0, -1) != 0;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    for (long long r = threadIdx.x; r < taken_before; r += kThreads) {
      const int page = k.free_pages[height - 1 - r];
      if (page >= 0 && page < k.pages) atomicCAS(&k.refs[page], -1, 0);
    }
    return;
  }
  for (long long i = threadIdx.x >> 5; i < n; i += kWarps) {
    const long long slot = sequences != nullptr ? sequences[i] : i;
    const bool copied = plan[i] < 0;
    const int taken = copied ? -plan[i] - 1 : plan[i];
    const int base = (k.lengths[slot] + k.page - 1) / k.page - (copied ? 1 : 0);
    for (int m = lane; m < taken; m += 32) {
      const int page = k.free_pages[height - 1 - firsts[i] - m];
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

// The first block of the cluster does the book; then, where there is more than
// one, all of them the copies (else a kernel behind this one does).
__global__ void __launch_bounds__(kThreads) extend_kernel(const __grid_constant__ cb_page_book k,
                                                          const __grid_constant__ cb_page_pools p, const int* counts,
                                                          const int* sequences, long long n, void* scratch, int* flag) {
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0) extend_book(k, counts, sequences, n, scratch, flag);
  if (gridDim.x == 1) return;
  cluster_sync();
  const Copies c = copies_of(scratch, n);
  copy_units(p, c.source, c.target, __ldcg(c.count), blockIdx.x * kWarps + threadIdx.x / 32, gridDim.x * kWarps, flag);
}

// Each pair by itself: all of it, or where it is refused none.
__global__ void __launch_bounds__(256) fork_kernel(cb_page_book k, const int* parents, const int* children,
                                                   long long n, int* flag) {
  pdl_launch_dependents();
  pdl_wait();
  const long long i = blockIdx.x;
  const int parent = parents[i], child = children[i];
  bool bad = parent < 0 || parent >= k.slots || child < 0 || child >= k.slots;
  for (long long j = threadIdx.x; j < n; j += blockDim.x)
    bad = bad || (j != i && children[j] == child) || parents[j] == child;
  const int length = bad ? 0 : k.lengths[parent];
  if (!bad) bad = k.lengths[child] != 0 || length < 0 || length > k.columns * k.page;
  for (long long m = threadIdx.x; !bad && m * k.page < length; m += blockDim.x) {
    const int page = k.table[parent * k.columns + m];
    bad = page < 0 || page >= k.pages;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    return;
  }
  for (long long m = threadIdx.x; m < k.columns; m += blockDim.x) {
    const int page = k.table[parent * k.columns + m];
    k.table[child * k.columns + m] = page;
    if (m * k.page < length) atomicAdd(&k.refs[page], 1);
  }
  __syncthreads();  // every thread has seen the child empty
  if (threadIdx.x == 0) k.lengths[child] = length;
}

// Entry e = i * columns + m of the call is dropped where need <= m < have of
// slot i.  A page that nobody holds any more is claimed by the last of its
// dropped entries: refs[page] goes from 0 to -(e + 1), the least of them.
// Each block of the cluster takes a contiguous range of the entries, in
// descending order; a thread keeps the pages of its first kKept entries.
constexpr int kKept = 4;

__global__ void __launch_bounds__(kThreads) truncate_kernel(cb_page_book k, const int* counts, const int* sequences,
                                                            int n, int* flag) {
  __shared__ long long shared[kWarps], first[kMostBlocks], second[kMostBlocks], third[kMostBlocks];
  cluster_begun();
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group group = cg::this_cluster();
  const int blocks = static_cast<int>(group.num_blocks()), rank = static_cast<int>(group.block_rank());
  const int columns = static_cast<int>(k.columns), entries = n * columns;
  const int height = *k.height;
  bool bad = height < 0 || height > k.pages;
  for (int i = threadIdx.x; i < n; i += kThreads) {  // every block for itself
    const int slot = sequences != nullptr ? sequences[i] : i;
    if (slot < 0 || slot >= k.slots) {
      bad = true;
      continue;
    }
    const int length = k.lengths[slot];
    bad = bad || length < 0 || length > k.columns * k.page ||
          (counts != nullptr && (counts[i] < 0 || counts[i] > length));
    for (int j = 0; j < i && sequences != nullptr; ++j) bad = bad || sequences[j] == slot;
  }
  const int per = ((entries + blocks - 1) / blocks + kThreads - 1) / kThreads * kThreads;
  const int begin = rank * per, end = min(begin + per, entries);
  auto entry = [&](int f) { return entries - 1 - f; };
  auto place = [&](int e) -> int* {  // of a dropped entry in the table
    const int i = e / columns, m = e % columns;
    const int slot = sequences != nullptr ? sequences[i] : i;
    const int length = k.lengths[slot], rest = counts != nullptr ? length - counts[i] : 0;
    const long long token = static_cast<long long>(m) * k.page;
    return token < length && token >= rest ? k.table + slot * k.columns + m : nullptr;
  };
  auto page_of = [&](int f) {
    const int* at = f < end ? place(entry(f)) : nullptr;
    if (at == nullptr) return -1;
    return *at < 0 || *at >= k.pages ? -2 : *at;
  };
  if (__syncthreads_or(bad)) {  // the same in every block
    if (threadIdx.x == 0) raise_flag(flag, CB_FLAG_BOOK);
    return;
  }
  int pages[kKept];
  for (int it = 0, f = begin + threadIdx.x; f < end; ++it, f += kThreads) {
    const int page = page_of(f);
    if (it < kKept) {
#pragma unroll
      for (int n = 0; n < kKept; ++n) pages[n] = n == it ? page : pages[n];
    }
    if (page >= 0) atomicSub(&k.refs[page], 1);
    if (page == -2) raise_flag(flag, CB_FLAG_BOOK);
  }
  auto known = [&](int it, int f) {
    int page = -1;
#pragma unroll
    for (int n = 0; n < kKept; ++n) page = n == it ? pages[n] : page;
    return it < kKept ? page : page_of(f);
  };
  long long total;
  cluster_all_begun();
  cluster_scan(0, first, &total);  // all are counted down
  for (int it = 0, f = begin + threadIdx.x; f < end; ++it, f += kThreads) {
    const int page = known(it, f);
    if (page >= 0 && __ldcg(&k.refs[page]) <= 0) atomicMin(&k.refs[page], -(entry(f) + 1));
  }
  cluster_scan(0, second, &total);  // all claims are in
  int mine = 0;
  for (int it = 0, f = begin + threadIdx.x; f < end; ++it, f += kThreads) {
    const int page = known(it, f);
    mine += page >= 0 && __ldcg(&k.refs[page]) == -(entry(f) + 1);
  }
  long long count;
  block_scan(mine, shared, &count);
  long long pushed = height + cluster_scan(count, third, &total);
  for (int at = begin; at < end; at += kThreads) {
    const int f = at + threadIdx.x, page = f < end ? known((at - begin) / kThreads, f) : -1;
    const bool claimed = page >= 0 && __ldcg(&k.refs[page]) == -(entry(f) + 1);
    long long sum;
    const long long to = pushed + block_scan(claimed, shared, &sum);
    if (claimed) {
      if (to < k.pages) k.free_pages[to] = page;
      else raise_flag(flag, CB_FLAG_BOOK);
      k.refs[page] = 0;
    }
    if (f < end) {
      int* gone = place(entry(f));
      if (gone != nullptr) *gone = -1;
    }
    pushed += sum;
  }
  cluster_sync();  // every block has used the lengths
  if (rank == 0) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int slot = sequences != nullptr ? sequences[i] : i;
      k.lengths[slot] = counts != nullptr ? k.lengths[slot] - counts[i] : 0;
    }
    if (threadIdx.x == 0) *k.height = static_cast<int>(height + total < k.pages ? height + total : k.pages);
  }
}

__global__ void __launch_bounds__(kThreads) compact_kernel(cb_page_book k, void* scratch, int* flag) {
  __shared__ long long shared[kWarps], first[kMostBlocks], second[kMostBlocks], third[kMostBlocks];
  cluster_begun();
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group group = cg::this_cluster();
  const int blocks = static_cast<int>(group.num_blocks()), rank = static_cast<int>(group.block_rank());
  const int pages = static_cast<int>(k.pages), thread = rank * kThreads + threadIdx.x, threads = blocks * kThreads;
  const Copies copies = copies_of(scratch, k.pages);
  int* to = copies.more;
  const int per = ((pages + blocks - 1) / blocks + kThreads - 1) / kThreads * kThreads;
  const int begin = rank * per, end = min(begin + per, pages);
  int live = 0;
  for (int p = begin + threadIdx.x; p < end; p += kThreads) {
    to[p] = p;
    live += k.refs[p] > 0;
  }
  long long sum, held;
  block_scan(live, shared, &sum);
  cluster_all_begun();
  cluster_scan(sum, first, &held);
  long long pair = 0;  // pages that move, holes
  for (int p = begin + threadIdx.x; p < end; p += kThreads) {
    const bool used = k.refs[p] > 0;
    pair += (static_cast<long long>(p >= held && used) << 32) + (p < held && !used);
  }
  block_scan(pair, shared, &sum);
  long long all;
  long long before = cluster_scan(sum, second, &all);
  const int moves = static_cast<int>(all >> 32);
  for (int at = begin; at < end; at += kThreads) {
    const int p = at + threadIdx.x;
    const bool used = p < end && k.refs[p] > 0, move = used && p >= held, hole = p < end && !used && p < held;
    const long long rank_of = before + block_scan((static_cast<long long>(move) << 32) + hole, shared, &sum);
    if (hole) copies.target[rank_of & 0xffffffffll] = p;
    if (move) copies.source[rank_of >> 32] = p;
    before += sum;
  }
  cluster_scan(0, third, &sum);  // the lists are written
  for (int r = thread; r < moves; r += threads) {
    const int source = __ldcg(copies.source + r), target = __ldcg(copies.target + r);
    to[source] = target;
    k.refs[target] = k.refs[source];
    k.refs[source] = 0;
  }
  cluster_sync();
  for (long long e = thread; e < k.slots * k.columns; e += threads) {
    const int page = k.table[e];
    if (page >= pages) raise_flag(flag, CB_FLAG_BOOK);
    else if (page >= held) k.table[e] = __ldcg(to + page);
  }
  for (int i = thread; i < pages - held; i += threads) k.free_pages[i] = pages - 1 - i;
  if (thread == 0) {
    *k.height = static_cast<int>(pages - held);
    *copies.count = moves;
  }
}

int book_check(const cb_page_book* k, long long n, const char* who) {
  CB_REQUIRE(k != nullptr && k->table && k->lengths && k->refs && k->free_pages && k->height, "%s: a null pointer", who);
  CB_REQUIRE(k->slots >= 1 && k->columns >= 1 && k->pages >= 1 && k->page >= 1, "%s: an empty book", who);
  // (entries are counted in 32 bits and rounded up to a multiple of a cluster's threads)
  CB_REQUIRE(k->columns * k->page < (1LL << 31) &&
                 k->slots * k->columns <= (1LL << 31) - kMostBlocks * kThreads * 2 &&
                 k->pages <= (1LL << 31) - kMostBlocks * kThreads * 2,
             "%s: %lld slots of %lld columns, %lld pages", who, k->slots, k->columns, k->pages);
  CB_REQUIRE(n >= 0 && n <= k->slots, "%s: %lld of %lld slots", who, n, k->slots);
  return CB_OK;
}

int pools_check(const cb_page_pools* p, const char* who) {
  CB_REQUIRE(p != nullptr && p->k_pages && p->v_pages && p->k_scale && p->v_scale, "%s: a null pointer", who);
  CB_REQUIRE(p->layers >= 1 && p->layers < (1 << 20) && p->pages >= 1 && p->pages < (1LL << 31) &&
                 p->page_bytes < (1LL << 31) && p->kv_heads >= 1 && p->page_bytes > 0 && p->page_bytes % 16 == 0,
             "%s: %lld layers of %lld pages of %lld bytes", who, p->layers, p->pages, p->page_bytes);
  CB_REQUIRE(reinterpret_cast<uintptr_t>(p->k_pages) % 16 == 0 && reinterpret_cast<uintptr_t>(p->v_pages) % 16 == 0,
             "%s: the pools must be 16-byte aligned", who);
  return CB_OK;
}

int launch_copies(const cb_page_pools& p, const int* source, const int* target, const int* count, long long most,
                  bool behind, int* flag, cudaStream_t stream) {
  const long long blocks = (most * p.layers * 2 + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  const long long cap = 1LL * (2048 / kCopyThreads) * sm_count();
  launch(copy_kernel, dim3(static_cast<unsigned>(blocks < cap ? blocks : cap)), dim3(kCopyThreads), 0, stream, behind, p,
         source, target, count, static_cast<int>(most), flag);
  return check_launch("cb_pages: copies");
}

// One cluster for `work` list entries: a block for each kThreads of them, up
// to eight.
template <typename... Expected, typename... Args>
int launch_cluster(void (*kernel)(Expected...), const char* what, long long work, cudaStream_t stream, Args... args) {
  unsigned blocks = 1;
  while (blocks < kMostBlocks && work > 1LL * kThreads * blocks) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<Expected>(args)...);
  return check_launch(what);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_pages_scratch(const cb_page_book* book, long long n) {
  if (book_check(book, n, "cb_pages_scratch") != CB_OK) return 0;
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
  // few bytes at most: one cluster does book and copies, in one launch (2.7 us
  // less for the host).  Its eight SMs copy at about 1 TB/s: with 16 slots' open
  // pages of 22 layers (5.8 MB read and written) fork and extend took 19.2 us that
  // way and 12.5 by a grid of their own, so that takes over at kClusterCopy.
  const bool together = 2LL * n * pools->layers * pools->page_bytes <= kClusterCopy;
  status = launch_cluster(extend_kernel, "cb_pages_extend", together ? 1LL * kMostBlocks * kThreads : 1, s, *book, *pools,
                          counts, sequences, n, scratch, error_flag);
  if (status != CB_OK || together) return status;
  const Copies c = copies_of(scratch, n);
  return launch_copies(*pools, c.source, c.target, c.count, n, true, error_flag, s);
}

int cb_pages_fork(const cb_page_book* book, const int* parents, const int* children, long long n, int* error_flag,
                  cb_stream_t stream) {
  const int status = book_check(book, n, "cb_pages_fork");
  if (status != CB_OK) return status;
  if (n == 0) return CB_OK;
  CB_REQUIRE(parents != nullptr && children != nullptr, "cb_pages_fork: a null pointer");
  launch(fork_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0, static_cast<cudaStream_t>(stream), true, *book,
         parents, children, n, error_flag);
  return check_launch("cb_pages_fork");
}

int cb_pages_truncate(const cb_page_book* book, const int* counts, const int* sequences, long long n, int* error_flag,
                      cb_stream_t stream) {
  const int status = book_check(book, n, "cb_pages_truncate");
  if (status != CB_OK) return status;
  if (n == 0) return CB_OK;
  return launch_cluster(truncate_kernel, "cb_pages_truncate", n * book->columns, static_cast<cudaStream_t>(stream),
                        *book, counts, sequences, n, error_flag);
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
  const long long entries = book->slots * book->columns;
  status = launch_cluster(compact_kernel, "cb_pages_compact", book->pages > entries ? book->pages : entries, s, *book,
                          scratch, error_flag);
  if (status != CB_OK) return status;
  const Copies c = copies_of(scratch, book->pages);
  return launch_copies(*pools, c.source, c.target, c.count, book->pages, true, error_flag, s);
}

int cb_pages_copy(const cb_page_pools* pools, const int* source, const int* target, long long n, int* error_flag,
                  cb_stream_t stream) {
  const int status = pools_check(pools, "cb_pages_copy");
  if (status != CB_OK) return status;
  CB_REQUIRE(n >= 0 && n < (1LL << 31), "cb_pages_copy: %lld pages", n);
  if (n == 0) return CB_OK;
  CB_REQUIRE(source != nullptr && target != nullptr, "cb_pages_copy: a null pointer");
  return launch_copies(*pools, source, target, nullptr, n, false, error_flag, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
