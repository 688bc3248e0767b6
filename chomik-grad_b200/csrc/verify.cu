// Verification of drafted tokens: cb_verify_draft.
//
// Speculative sampling keeps the target's distribution: token t is accepted
// with probability min(1, p_t(x_t) / q_t(x_t)), tested as u q < p, and at the
// first refusal the replacement is drawn from max(p - q, 0), normalised.  The
// draw is by inverse cumulative sum over fixed-point weights, so the sums are
// exact in any order and the token does not depend on how the row is split.
//
// One block per sequence.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ unsigned long long fixed_point(float x) {
  // float -> integer conversion truncates; NaN and negative numbers weigh nothing
  return x > 0.0f ? static_cast<unsigned long long>(fminf(x, 1.0f) * 1099511627776.0f) : 0ull;
}

__device__ __forceinline__ unsigned long long warp_inclusive(unsigned long long v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, v, o);
    if (static_cast<int>(threadIdx.x & 31) >= o) v += up;
  }
  return v;
}

// Exclusive sum in thread order, and the block's sum.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* shared,
                                                         unsigned long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned long long incl = warp_inclusive(v);
  __syncthreads();
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  if (warp == 0) shared[lane] = warp_inclusive(shared[lane]);
  __syncthreads();
  *total = shared[kWarps - 1];
  return incl - v + (warp > 0 ? shared[warp - 1] : 0);
}

__global__ void __launch_bounds__(kThreads) verify_kernel(cb_verify_args a) {
  __shared__ unsigned long long shared[kWarps];
  const long long b = blockIdx.x;
  long long n = a.counts != nullptr ? a.counts[b] : a.tokens;
  if (n < 0 || n > a.tokens) {
    if (threadIdx.x == 0) raise_flag(a.error_flag, CB_FLAG_BOOK);
    n = n < 0 ? 0 : a.tokens;
  }
  const long long* drafted = a.drafted + b * a.tokens;
  const double* u = a.uniforms + b * (a.tokens + 1);
  long long accepted = 0;
  for (; accepted < n; ++accepted) {
    const long long x = drafted[accepted];
    if (x < 0 || x >= a.vocab) {
      if (threadIdx.x == 0) raise_flag(a.error_flag, CB_FLAG_INDEX);
      break;
    }
    const float p = load_as_f32(a.target, b * a.target_strides[0] + accepted * a.target_strides[1] + x, a.dtype);
    const float q = load_as_f32(a.draft, b * a.draft_strides[0] + accepted * a.draft_strides[1] + x, a.dtype);
    if (!(u[accepted] * static_cast<double>(q) < static_cast<double>(p))) break;
  }
  const bool refused = accepted < n;
  const long long p_row = b * a.target_strides[0] + accepted * a.target_strides[1];
  const long long q_row = b * a.draft_strides[0] + accepted * a.draft_strides[1];
  unsigned long long rest = 0, whole = 0;
  bool nan = false;
  for (long long j = threadIdx.x; j < a.vocab; j += kThreads) {
    const float p = load_as_f32(a.target, p_row + j, a.dtype);
    const float q = refused ? load_as_f32(a.draft, q_row + j, a.dtype) : 0.0f;
    nan = nan || p != p || q != q;
    rest += fixed_point(p - q);
    whole += fixed_point(p);
  }
  nan = __syncthreads_or(nan);
  unsigned long long rest_total, whole_total;
  block_scan(rest, shared, &rest_total);
  block_scan(whole, shared, &whole_total);
  const bool from_rest = rest_total > 0;
  const unsigned long long total = from_rest ? rest_total : whole_total;
  __shared__ long long token;
  if (threadIdx.x == 0) token = -1;
  __syncthreads();
  if (!nan && total > 0) {
    long long bar = static_cast<long long>(u[a.tokens] * static_cast<double>(total));
    if (bar > static_cast<long long>(total) - 1) bar = static_cast<long long>(total) - 1;
    unsigned long long before = 0;
    for (long long at = 0; at < a.vocab; at += kThreads) {
      const long long j = at + threadIdx.x;
      unsigned long long w = 0;
      if (j < a.vocab) {
        const float p = load_as_f32(a.target, p_row + j, a.dtype);
        const float q = refused && from_rest ? load_as_f32(a.draft, q_row + j, a.dtype) : 0.0f;
        w = fixed_point(p - q);
      }
      unsigned long long sum;
      const unsigned long long lower = before + block_scan(w, shared, &sum);
      const unsigned long long limit = static_cast<unsigned long long>(bar);
      if (lower <= limit && limit < lower + w) token = j;
      before += sum;
      if (before > limit) break;  // the same for every thread
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.accepted[b] = static_cast<int>(accepted);
    if (token < 0) raise_flag(a.error_flag, CB_FLAG_NAN);
  }
  for (long long t = threadIdx.x; t <= a.tokens; t += kThreads)
    a.out[b * (a.tokens + 1) + t] = t < accepted ? drafted[t] : t == accepted ? token : -1;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_verify_draft(const cb_verify_args* args, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_verify_draft: null arguments");
  const cb_verify_args& a = *args;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_verify_draft: probabilities must be float32, bfloat16 or float16");
  CB_REQUIRE(a.batch >= 0 && a.batch < (1LL << 31) && a.tokens >= 0 && a.tokens < (1LL << 20),
             "cb_verify_draft: %lld sequences of %lld tokens", a.batch, a.tokens);
  // 2^40 * vocab stays inside 63 bits
  CB_REQUIRE(a.vocab >= 1 && a.vocab <= (1LL << 22), "cb_verify_draft: vocabulary of %lld", a.vocab);
  if (a.batch == 0) return CB_OK;
  CB_REQUIRE(a.target && a.uniforms && a.accepted && a.out && (a.tokens == 0 || (a.draft && a.drafted)),
             "cb_verify_draft: a null pointer");
  verify_kernel<<<static_cast<unsigned>(a.batch), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("cb_verify_draft");
}
