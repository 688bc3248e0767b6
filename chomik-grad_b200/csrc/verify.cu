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
// block that holds the threshold reads the run that does again (some KB, from
// L2) to find the token.  What bounds it: one target row and, where a draft was
// refused, one draft row per sequence; in small batches the chain of dependent
// loads (drafted token, its probabilities, the rows).  Measured: 64 rows of 7
// drafts and 128,256 float32 probabilities 18.0 us (2 us until the rows, which
// take until 9 to 14, the exchange until 13 to 15, the second read 1.5), one
// row of 4 drafts and 32,000 4.6 us.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostBlocks = 8;  // of a cluster: the portable limit

using u64 = unsigned long long;

// trunc(min(max(x, 0), 1) * 2^40), NaN gives 0, as hi * 2^23 + lo: adding 2^23
// with rounding toward zero leaves the integer part in the low bits of the sum
// (float32 instructions only; a 64-bit conversion takes some ten times as long).
// The bits of 2^23 itself are left in both for the caller to take off.
constexpr uint32_t kBias = 0x4b000000u;
__device__ __forceinline__ void fixed_parts(float x, uint32_t& hi, uint32_t& lo) {
  const float big = 8388608.0f, y = fminf(fmaxf(x, 0.0f), 1.0f) * 131072.0f;
  const float t = __fadd_rz(y, big);
  hi = __float_as_uint(t);
  lo = __float_as_uint(__fadd_rz((y - (t - big)) * big, big));
}
__device__ __forceinline__ u64 fixed_point(float x) {
  uint32_t hi, lo;
  fixed_parts(x, hi, lo);
  return (static_cast<u64>(hi - kBias) << 23) + (lo - kBias);
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

template <int DT>
__device__ __forceinline__ void unpack(const uint4& w, float* x) {
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
}

// kPer probabilities from element j of a row of `vocab`; those past its end are 0.
template <int DT>
__device__ __forceinline__ void load_row(const char* row, long long j, long long vocab, bool wide, float* x) {
  constexpr int kPer = Item<DT>::kPer;
  if (wide && j + kPer <= vocab) {
    unpack<DT>(*reinterpret_cast<const uint4*>(row + j * (16 / kPer)), x);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = j + i < vocab ? load_as_f32(row, j + i, DT) : 0.0f;
  }
}

struct Sums {  // of one block
  u64 weight;
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
  __shared__ Sums warps[kWarps], cluster[2][kMostBlocks];
  __shared__ u64 parts[kWarps];
  cluster_begun();
  pdl_launch_dependents();
  pdl_wait();
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

  // 1. sums of the runs.  The remainders p - q first; only where a refused
  // draft leaves none, the target's own probabilities (`second`).
  cg::cluster_group group = cg::this_cluster();
  u64 total = 0, before = 0;
  bool second = false;
  int bad = 0;
  for (;;) {
    const bool with_draft = refused && !second;
    u64 sum = 0;
    uint32_t hi = 0, lo = 0;
    int held = 0;  // steps summed in hi and lo
    bool nan = false;
    auto flush = [&] {
      const uint32_t bias = static_cast<uint32_t>(held) * kPer * kBias;
      sum += (static_cast<u64>(hi - bias) << 23) + (lo - bias);
      hi = lo = 0;
      held = 0;
    };
    auto add = [&](const float* p, const float* q) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float other = with_draft ? q[i] : 0.0f;
        nan = nan || p[i] != p[i] || other != other;
        uint32_t h, l;
        fixed_parts(p[i] - other, h, l);
        hi += h;
        lo += l;
      }
      if (++held == 32) flush();  // 32 steps of up to 8 weights below 2^23: their sum is below 2^32
    };
    constexpr int kStep = 32 * kPer, kBatch = 4;  // elements of a warp's loads; of them in flight
    long long first = from;
    for (; wide && first + kBatch * kStep <= to; first += kBatch * kStep) {
      uint4 p[kBatch], q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) p[i] = reinterpret_cast<const uint4*>(p_row)[(first + i * kStep) / kPer + lane];
      if (with_draft) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) q[i] = reinterpret_cast<const uint4*>(q_row)[(first + i * kStep) / kPer + lane];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        float x[kPer], y[kPer];
        unpack<DT>(p[i], x);
        if (with_draft) unpack<DT>(q[i], y);
        add(x, y);
      }
    }
    for (; first < to; first += kStep) {
      float x[kPer], y[kPer];
      load_row<DT>(p_row, first + lane * kPer, a.vocab, wide, x);
      if (with_draft) load_row<DT>(q_row, first + lane * kPer, a.vocab, wide, y);
      add(x, y);
    }
    flush();
    sum = warp_total(sum);
    nan = __any_sync(0xffffffffu, nan);
    if (lane == 0) warps[warp] = {sum, nan};
    __syncthreads();
    if (!second) cluster_all_begun();
    if (static_cast<int>(threadIdx.x) < blocks) {  // a copy of the block's sums for each block of the cluster
      Sums mine = {0, 0};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mine.weight += warps[w].weight;
        mine.nan |= warps[w].nan;
      }
      *group.map_shared_rank(&cluster[second][rank], threadIdx.x) = mine;
    }
    cluster_sync();
    total = 0;
    for (int r = 0; r < blocks; ++r) {
      if (r == rank) before = total;
      total += cluster[second][r].weight;
      bad |= cluster[second][r].nan;
    }
    if (total > 0 || !with_draft || bad) break;  // the same in every block
    second = true;
  }

  // 2. the threshold, and the warp that holds it
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
  if (bad || bar < before || bar >= before + cluster[second][rank].weight) return;  // the same in the block

  // 3. the block that holds it reads that warp's run once more, each thread a
  // contiguous part, and the thread whose part holds it finds the token
  int holder = 0;
  while (bar >= before + warps[holder].weight) before += warps[holder++].weight;
  const bool with_draft = refused && !second;
  auto weights = [&](long long j, u64* w) {
    float p[kPer], q[kPer];
    load_row<DT>(p_row, j, a.vocab, wide, p);
    if (with_draft) load_row<DT>(q_row, j, a.vocab, wide, q);
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      w[i] = fixed_point(p[i] - (with_draft ? q[i] : 0.0f));
      sum += w[i];
    }
    return sum;
  };
  const long long start = (static_cast<long long>(rank) * kWarps + holder) * run;
  const long long part = (run / kPer + kThreads - 1) / kThreads * kPer;
  const long long begin = start + threadIdx.x * part, end = begin + part < start + run ? begin + part : start + run;
  u64 w[kPer], sum = 0;
#pragma unroll 4
  for (long long j = begin; j < end; j += kPer) sum += weights(j, w);
  u64 upto = sum;  // inclusive sum over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 31) parts[warp] = upto;
  __syncthreads();
  u64 running = before + upto - sum;
  for (int p = 0; p < warp; ++p) running += parts[p];
  if (bar < running || bar >= running + sum) return;
  for (long long j = begin; j < end; j += kPer) {  // one thread
    weights(j, w);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (running <= bar && bar < running + w[i]) a.out[b * (a.tokens + 1) + accepted] = j + i;
      running += w[i];
    }
  }
}

template <int DT>
int launch_verify(const cb_verify_args& a, cudaStream_t stream) {
  // blocks of a row: as few as leave a thread 16 elements
  int blocks = 1;
  while (blocks < kMostBlocks && a.vocab > 16LL * kThreads * blocks) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(blocks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
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
