// Verification of drafted tokens: cb_verify_draft.
//
// Speculative sampling keeps the target's distribution: token t is accepted
// with probability min(1, p_t(x_t) / q_t(x_t)), tested as u q < p, and at the
// first refusal the replacement is drawn from max(p - q, 0), normalised.  The
// draw is by inverse cumulative sum over fixed-point weights, so the sums are
// exact in any order and the token does not depend on how the row is split.
//
// One cluster of blocks per sequence, one launch.  A row is read once: a warp
// owns a contiguous run of it, the warps' sums are joined over the block, and
// the blocks' over the cluster through distributed shared memory; then the
// warp whose run holds the threshold reads its run again (some KB, from L2) to
// find the token.  What bounds it: one target row and, where a draft was
// refused, one draft row per sequence; in small batches the chain of dependent
// loads (drafted token, its probabilities, the rows).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostBlocks = 8;  // of a cluster: the portable limit

using u64 = unsigned long long;

__device__ __forceinline__ u64 fixed_point(float x) {
  // float -> integer conversion truncates; NaN and negative numbers weigh nothing
  return x > 0.0f ? static_cast<u64>(fminf(x, 1.0f) * 1099511627776.0f) : 0ull;
}

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int DT>
struct Item {
  static constexpr int kPer = DT == CB_F32 ? 4 : 8;  // elements of 16 bytes
};

// kPer probabilities from element j of a row of `vocab`; those past its end are 0.
template <int DT>
__device__ __forceinline__ void load_row(const char* row, long long j, long long vocab, bool wide, float* x) {
  constexpr int kPer = Item<DT>::kPer;
  if (wide && j + kPer <= vocab) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + j * (16 / kPer));
    if (DT == CB_F32) {
      x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y);
      x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    } else if (DT == CB_BF16) {
      unpack_bf16x8(w, x);
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __low2float(h[i]);
        x[2 * i + 1] = __high2float(h[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = j + i < vocab ? load_as_f32(row, j + i, DT) : 0.0f;
  }
}

struct Sums {  // of one block
  u64 rest, whole;
  int nan;
};

// Elements of a warp's run: `blocks` blocks cover the vocabulary, in whole
// steps of 32 lanes.
__host__ __device__ __forceinline__ long long run_of(long long vocab, int blocks, int per) {
  const long long step = 32LL * per, warps = 1LL * blocks * kWarps;
  return ((vocab + warps - 1) / warps + step - 1) / step * step;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ cb_verify_args a, int blocks) {
  constexpr int kPer = Item<DT>::kPer, kItem = 16 / kPer;
  __shared__ Sums warps[kWarps], cluster[kMostBlocks];
  cluster_begun();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = static_cast<int>(blockIdx.x) % blocks;
  const long long b = blockIdx.x / blocks;
  long long n = a.counts != nullptr ? a.counts[b] : a.tokens;
  if (n < 0 || n > a.tokens) {
    if (threadIdx.x == 0) raise_flag(a.error_flag, CB_FLAG_BOOK);
    n = n < 0 ? 0 : a.tokens;
  }
  const long long* drafted = a.drafted + b * a.tokens;
  const double* u = a.uniforms + b * (a.tokens + 1);
  const double last = u[a.tokens];
  const char* target = static_cast<const char*>(a.target) + b * a.target_strides[0] * kItem;
  const char* draft = static_cast<const char*>(a.draft) + b * a.draft_strides[0] * kItem;
  long long accepted = n;
  for (long long first = 0; first < n; first += 32) {  // every warp for itself: a lane for each draft
    const long long t = first + lane;
    bool refused = false;
    if (t < n) {
      const long long x = drafted[t];
      refused = true;
      if (x >= 0 && x < a.vocab) {
        const float p = load_as_f32(target, t * a.target_strides[1] + x, DT);
        const float q = load_as_f32(draft, t * a.draft_strides[1] + x, DT);
        refused = !(u[t] * static_cast<double>(q) < static_cast<double>(p));
      }
    }
    const unsigned who = __ballot_sync(0xffffffffu, refused);
    if (who != 0) {
      accepted = first + __ffs(who) - 1;
      break;
    }
  }
  const bool refused = accepted < n;
  if (refused && threadIdx.x == 0 && (drafted[accepted] < 0 || drafted[accepted] >= a.vocab))
    raise_flag(a.error_flag, CB_FLAG_INDEX);
  const char* p_row = target + accepted * a.target_strides[1] * kItem;
  const char* q_row = draft + accepted * a.draft_strides[1] * kItem;
  const bool wide = (reinterpret_cast<uintptr_t>(p_row) | (refused ? reinterpret_cast<uintptr_t>(q_row) : 0)) % 16 == 0;
  const long long run = run_of(a.vocab, blocks, kPer);
  const long long from = (static_cast<long long>(rank) * kWarps + warp) * run;
  const long long to = from + run < a.vocab ? from + run : a.vocab;

  // 1. sums of the runs
  u64 rest = 0, whole = 0;
  bool nan = false;
#pragma unroll 4
  for (long long j = from + lane * kPer; j < to; j += 32 * kPer) {
    float p[kPer], q[kPer];
    load_row<DT>(p_row, j, a.vocab, wide, p);
    if (refused) load_row<DT>(q_row, j, a.vocab, wide, q);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float other = refused ? q[i] : 0.0f;
      nan = nan || p[i] != p[i] || other != other;
      rest += fixed_point(p[i] - other);
      whole += fixed_point(p[i]);
    }
  }
  rest = warp_total(rest);
  whole = warp_total(whole);
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) warps[warp] = {rest, whole, nan};
  __syncthreads();
  cg::cluster_group group = cg::this_cluster();
  cluster_all_begun();
  if (static_cast<int>(threadIdx.x) < blocks) {  // a copy of the block's sums for each block of the cluster
    Sums mine = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mine.rest += warps[w].rest;
      mine.whole += warps[w].whole;
      mine.nan |= warps[w].nan;
    }
    *group.map_shared_rank(&cluster[rank], threadIdx.x) = mine;
  }
  group.sync();

  // 2. the threshold, and the warp that holds it
  u64 rest_total = 0, whole_total = 0, rest_before = 0, whole_before = 0;
  int bad = 0;
  for (int r = 0; r < blocks; ++r) {
    if (r == rank) {
      rest_before = rest_total;
      whole_before = whole_total;
    }
    rest_total += cluster[r].rest;
    whole_total += cluster[r].whole;
    bad |= cluster[r].nan;
  }
  const bool from_rest = rest_total > 0;
  const u64 total = from_rest ? rest_total : whole_total;
  bad |= total == 0;
  u64 bar = 0;
  if (!bad) {
    const long long scaled = static_cast<long long>(last * static_cast<double>(total));
    bar = static_cast<u64>(scaled < static_cast<long long>(total) - 1 ? scaled : static_cast<long long>(total) - 1);
    bad = scaled < 0;  // a uniform number below zero
  }
  if (rank == 0) {
    if (threadIdx.x == 0) {
      a.accepted[b] = static_cast<int>(accepted);
      if (bad) raise_flag(a.error_flag, CB_FLAG_NAN);
    }
    for (long long t = threadIdx.x; t <= a.tokens; t += kThreads)
      if (t != accepted || bad) a.out[b * (a.tokens + 1) + t] = t < accepted ? drafted[t] : -1;
  }
  if (bad) return;
  u64 before = from_rest ? rest_before : whole_before;
  for (int w = 0; w < warp; ++w) before += from_rest ? warps[w].rest : warps[w].whole;
  const u64 mine = from_rest ? warps[warp].rest : warps[warp].whole;
  if (bar < before || bar >= before + mine) return;

  // 3. that warp's run once more, in order
  for (long long first = from; first < to; first += 32 * kPer) {
    float p[kPer], q[kPer];
    load_row<DT>(p_row, first + lane * kPer, a.vocab, wide, p);
    if (refused && from_rest) load_row<DT>(q_row, first + lane * kPer, a.vocab, wide, q);
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += fixed_point(p[i] - (refused && from_rest ? q[i] : 0.0f));
    u64 upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    u64 running = before + upto - sum;
    if (running <= bar && bar < before + upto) {  // one lane
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const u64 w = fixed_point(p[i] - (refused && from_rest ? q[i] : 0.0f));
        if (running <= bar && bar < running + w) a.out[b * (a.tokens + 1) + accepted] = first + lane * kPer + i;
        running += w;
      }
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (before > bar) return;
  }
}

template <int DT>
int launch_verify(const cb_verify_args& a, cudaStream_t stream) {
  // blocks of a row: as few as leave a thread 16 elements (32000 of float32 by
  // four blocks: 4.9 us; by one: 8.5, by eight: 5.0)
  int blocks = 1;
  while (blocks < kMostBlocks && a.vocab > 16LL * kThreads * blocks) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(blocks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<DT>, a, blocks);
  return check_launch("cb_verify_draft");
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_verify_draft(const cb_verify_args* args, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_verify_draft: null arguments");
  const cb_verify_args& a = *args;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_verify_draft: probabilities must be float32, bfloat16 or float16");
  CB_REQUIRE(a.batch >= 0 && a.batch < (1LL << 28) && a.tokens >= 0 && a.tokens < (1LL << 20),
             "cb_verify_draft: %lld sequences of %lld tokens", a.batch, a.tokens);
  // 2^40 * vocab stays inside 63 bits
  CB_REQUIRE(a.vocab >= 1 && a.vocab <= (1LL << 22), "cb_verify_draft: vocabulary of %lld", a.vocab);
  if (a.batch == 0) return CB_OK;
  CB_REQUIRE(a.target && a.uniforms && a.accepted && a.out && (a.tokens == 0 || (a.draft && a.drafted)),
             "cb_verify_draft: a null pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == CB_F32) return launch_verify<CB_F32>(a, s);
  if (a.dtype == CB_BF16) return launch_verify<CB_BF16>(a, s);
  return launch_verify<CB_F16>(a, s);
}
