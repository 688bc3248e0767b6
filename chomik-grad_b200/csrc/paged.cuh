// Shared by the kernels over the paged 8-bit KV cache (cb_paged_cache).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace cb {

__device__ __forceinline__ void raise_flag(int* flag, int code) {
  if (flag != nullptr) atomicMax(flag, code);
}

// Cluster barriers without .aligned: threads of a warp may come to them one by
// one, out of loops and branches that ended at different times.
//
// A cluster's blocks write to one another's shared memory only once all have
// begun: each arrives first thing, and waits before its first such write.
__device__ __forceinline__ void cluster_begun() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_all_begun() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
// Orders the memory of all threads of the cluster, as __syncthreads that of a block.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

inline int paged_cache_check(const cb_paged_cache& c, const char* who) {
  CB_REQUIRE(c.storage == CB_I8 || c.storage == CB_E4M3, "%s: storage must be int8 or e4m3 (got code %d)", who,
             c.storage);
  CB_REQUIRE(c.head_size == 32 || c.head_size == 64 || c.head_size == 128,
             "%s: head_size must be 32, 64 or 128 (got %d)", who, c.head_size);
  CB_REQUIRE(c.page >= 16 && c.page <= 256 && (c.page & (c.page - 1)) == 0,
             "%s: page must be 16, 32, 64, 128 or 256 (got %d)", who, c.page);
  CB_REQUIRE(c.kv_heads >= 1 && c.kv_heads <= 32767, "%s: kv_heads %d", who, c.kv_heads);
  CB_REQUIRE(c.pages >= 1 && c.pages < (1LL << 31), "%s: %lld pages", who, c.pages);
  CB_REQUIRE(c.slots >= 1 && c.columns >= 1 && c.columns * c.page < (1LL << 31) && c.slots < (1LL << 31),
             "%s: %lld slots of %lld columns", who, c.slots, c.columns);
  CB_REQUIRE(c.k_pages && c.v_pages && c.k_scale && c.v_scale && c.table && c.lengths, "%s: a null pointer", who);
  CB_REQUIRE(reinterpret_cast<uintptr_t>(c.k_pages) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v_pages) % 16 == 0,
             "%s: the pools must be 16-byte aligned", who);
  return CB_OK;
}

// What sequence `b` of a call works on: its slot's table row, the tokens it
// holds and the new ones among them.  False (and CB_FLAG_BOOK) where the book
// or the call's lists name something outside the cache.
struct PagedRow {
  const int* table;
  int length, count;
};
__device__ __forceinline__ bool paged_row(const cb_paged_cache& c, const int* sequences, const int* counts,
                                          long long tokens, long long b, int* flag, PagedRow* row) {
  const long long slot = sequences != nullptr ? sequences[b] : b;
  if (slot < 0 || slot >= c.slots) {
    raise_flag(flag, CB_FLAG_BOOK);
    return false;
  }
  const int length = c.lengths[slot];
  const long long count = counts != nullptr ? counts[b] : tokens;
  if (count < 0 || count > tokens || length < count || length > c.columns * c.page) {
    raise_flag(flag, CB_FLAG_BOOK);
    return false;
  }
  row->table = c.table + slot * c.columns;
  row->length = length;
  row->count = static_cast<int>(count);
  return true;
}

}  // namespace cb
