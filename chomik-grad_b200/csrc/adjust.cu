// Penalties, biases and masks on logit rows before a token is chosen: cb_adjust_logits.
//
// For token v of a row with the history t_0 .. t_(n-1), of which the first
// `prompt` were given and the rest were made:
//   c = #{i < n: t_i = v},  d = #{prompt <= i < n: t_i = v}
//   x = l > 0 ? l / r : l * r  where c > 0, else l
//   x = x - (frequency * d + presence * [d > 0]) + sum of the biases of v
//   x = -inf where v's bit of the mask is clear
// in float32, rounded once to the logits' type.
//
// What bounds it: the logits are read and written once (2 * item bytes a token
// and 1/8 of the mask).  A block takes a slice of one row's vocabulary, with a
// counter for each of its tokens in shared memory, so that the history (read by
// every slice of the row, from L2) becomes counts without a pass over global
// memory; the slice's logits are loaded into registers before that, so that the
// two latencies overlap.  Biases are few: the thread of a token's first entry
// sums them in the list's order (no float atomics: equal inputs give equal bits),
// computes the token by itself and writes it after the slice.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kAdjustThreads = 512;
constexpr int kMaxBiases = 1024;
constexpr unsigned kSeen = 0x80000000u;  // of a counter: anywhere in the history; below it: made

struct AdjustPlan {
  cb_adjust_args a;
  int slices, slice;  // of a row, and their tokens
  int shared_lead;    // logits and out lie alike to 16 bytes in every row: wide accesses
};

struct Penalty {
  float repetition, frequency, presence;
};

__device__ __forceinline__ float adjusted(float x, unsigned count, const Penalty& p) {
  if (count != 0) {
    x = x > 0.0f ? x / p.repetition : x * p.repetition;
    const unsigned made = count & ~kSeen;
    if (made != 0) x -= p.frequency * static_cast<float>(made) + p.presence;
  }
  return x;
}

__device__ __forceinline__ bool is_allowed(const int* allowed, long long v) {
  return allowed == nullptr || (static_cast<unsigned>(allowed[v >> 5]) >> (v & 31) & 1u) != 0;
}

// Eight neighbouring elements: one 16-byte access for 16-bit types, two for float32.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  static constexpr int kCode = CB_F32;
  float x[8];
  __device__ __forceinline__ float get(int i) const { return x[i]; }
  __device__ __forceinline__ void set(int i, float v) { x[i] = v; }
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void store(float* p) const {
#pragma unroll
    for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
};
struct EightHalves {
  uint32_t w[4];
  __device__ __forceinline__ uint16_t half_of(int i) const { return static_cast<uint16_t>(w[i / 2] >> (i % 2 * 16)); }
  __device__ __forceinline__ void set_half(int i, uint16_t h) {
    w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | static_cast<uint32_t>(h) << 16 : (w[i / 2] & 0xffff0000u) | h;
  }
  __device__ __forceinline__ void load(const void* p) {
    const uint4 v = *static_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void store(void* p) const {
    *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Eight<__nv_bfloat16> : EightHalves {
  static constexpr int kCode = CB_BF16;
  __device__ __forceinline__ float get(int i) const { return bf16_bits_to_f32(half_of(i)); }
  __device__ __forceinline__ void set(int i, float v) { set_half(i, __bfloat16_as_ushort(__float2bfloat16_rn(v))); }
};
template <>
struct Eight<__half> : EightHalves {
  static constexpr int kCode = CB_F16;
  __device__ __forceinline__ float get(int i) const { return __half2float(__ushort_as_half(half_of(i))); }
  __device__ __forceinline__ void set(int i, float v) { set_half(i, __half_as_ushort(__float2half_rn(v))); }
};

// EIGHTS: runs of eight neighbouring tokens that a thread takes.
template <typename T, int EIGHTS>
__global__ void __launch_bounds__(kAdjustThreads) adjust_kernel(const __grid_constant__ AdjustPlan p) {
  constexpr int kSlice = kAdjustThreads * 8 * EIGHTS, kOwn = kMaxBiases / kAdjustThreads;
  extern __shared__ __align__(16) unsigned counts[];  // of the slice's tokens, where there is a history
  __shared__ int listed[kMaxBiases];                  // the biases' tokens, -1 for those outside the vocabulary
  const cb_adjust_args& a = p.a;
  const long long row = blockIdx.x / p.slices;
  const int thread = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();

  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.out_ld;
  // Places are counted from the last 16-byte boundary at or before the row's
  // beginning: token = place - lead.
  const int lead = p.shared_lead ? static_cast<int>(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T)) : 0;
  const long long first = static_cast<long long>(blockIdx.x % p.slices) * kSlice - lead;  // token of place 0
  const int* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_ld : nullptr;

  Eight<T> x[EIGHTS];
  auto token_of = [&](int n) { return first + (n * kAdjustThreads + thread) * 8; };
  auto whole = [&](long long v) { return p.shared_lead && v >= 0 && v + 8 <= a.vocab; };
#pragma unroll
  for (int n = 0; n < EIGHTS; ++n) {
    const long long v = token_of(n);
    if (whole(v)) {
      x[n].load(in + v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v + i >= 0 && v + i < a.vocab) x[n].set(i, load_as_f32(in, v + i, Eight<T>::kCode));
    }
  }
  Penalty penalty{a.repetition, a.frequency, a.presence};
  if (a.tokens != nullptr) {
    if (a.repetitions != nullptr) penalty.repetition = a.repetitions[row];
    if (a.frequencies != nullptr) penalty.frequency = a.frequencies[row];
    if (a.presences != nullptr) penalty.presence = a.presences[row];
    for (int i = thread; i < kSlice / 4; i += kAdjustThreads)
      reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
    long long length = a.lengths != nullptr ? a.lengths[row] : a.history;
    long long prompt = a.prompts != nullptr ? a.prompts[row] : 0;
    if (length < 0 || length > a.history || prompt < 0 || prompt > length) {
      raise_flag(a.error_flag, CB_FLAG_HISTORY);
      length = min(max(length, 0LL), a.history);
      prompt = min(max(prompt, 0LL), length);
    }
    __syncthreads();
    const long long at = row * a.token_ld;
#pragma unroll 4
    for (long long i = thread; i < length; i += kAdjustThreads) {
      const long long token = load_index(a.tokens, at + i, a.token_dtype);
      const long long place = token - first;
      if (token >= 0 && token < a.vocab && place >= 0 && place < kSlice) {
        if (i >= prompt) atomicAdd(counts + place, 1u);
        else atomicOr(counts + place, kSeen);
      }
    }
  }
  int patched[kOwn];
  float patch[kOwn];
  if (a.biases > 0) {
    for (int i = thread; i < a.biases; i += kAdjustThreads) {
      const long long v = load_index(a.bias_tokens, row * a.bias_token_ld + i, a.bias_token_dtype);
      listed[i] = v >= 0 && v < a.vocab ? static_cast<int>(v) : -1;
    }
  }
  __syncthreads();
  if (a.biases > 0) {
    const float* bias = a.bias + row * a.bias_ld;
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
      const int own = n * kAdjustThreads + thread;
      const int v = own < a.biases ? listed[own] : -1;
      const long long place = v - first;
      patched[n] = -1;
      if (v < 0 || place < 0 || place >= kSlice) continue;
      bool earlier = false;
      for (int i = 0; i < own; ++i) earlier = earlier || listed[i] == v;
      if (earlier) continue;
      float sum = bias[own];
      for (int i = own + 1; i < a.biases; ++i)
        if (listed[i] == v) sum += bias[i];
      patched[n] = v;
      patch[n] = adjusted(load_as_f32(in, v, Eight<T>::kCode), a.tokens != nullptr ? counts[place] : 0u, penalty) + sum;
      if (!is_allowed(allowed, v)) patch[n] = -INFINITY;
    }
    __syncthreads();  // the row's logits that the patches need are read: out may be the same memory
  }
#pragma unroll
  for (int n = 0; n < EIGHTS; ++n) {
    const long long v = token_of(n);
    if (v + 8 <= 0 || v >= a.vocab) continue;
    unsigned bits = 0xffu;
    if (allowed != nullptr) {
      bits = 0;
      const long long low = max(v, 0LL), word = low >> 5;
      const unsigned a0 = allowed[word], a1 = (word + 1) * 32 < a.vocab ? allowed[word + 1] : 0;
      bits = __funnelshift_r(a0, a1, static_cast<unsigned>(low & 31)) << static_cast<int>(low - v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float y = x[n].get(i);
      if (a.tokens != nullptr) y = adjusted(y, counts[(n * kAdjustThreads + thread) * 8 + i], penalty);
      x[n].set(i, (bits >> i & 1u) != 0 ? y : -INFINITY);
    }
    if (whole(v)) {
      x[n].store(out + v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v + i >= 0 && v + i < a.vocab) store_from_f32(out, v + i, Eight<T>::kCode, x[n].get(i));
    }
  }
  if (a.biases > 0) {
    __syncthreads();  // (the patches come after the slice)
#pragma unroll
    for (int n = 0; n < kOwn; ++n)
      if (patched[n] >= 0) store_from_f32(out, patched[n], Eight<T>::kCode, patch[n]);
  }
}

template <typename T, int EIGHTS>
int run_adjust(AdjustPlan p, cudaStream_t stream) {
  constexpr int kSlice = kAdjustThreads * 8 * EIGHTS;
  const long long item = sizeof(T);
  const uintptr_t in = reinterpret_cast<uintptr_t>(p.a.logits), out = reinterpret_cast<uintptr_t>(p.a.out);
  p.shared_lead = (in - out) % 16 == 0 && (p.a.rows == 1 || (p.a.ld - p.a.out_ld) * item % 16 == 0);
  p.slice = kSlice;
  const long long slices = (p.a.vocab + 7 + kSlice - 1) / kSlice;
  CB_REQUIRE(slices * p.a.rows < (1LL << 31), "cb_adjust_logits: %lld rows of %lld", p.a.rows, p.a.vocab);
  p.slices = static_cast<int>(slices);
  launch(adjust_kernel<T, EIGHTS>, dim3(static_cast<unsigned>(slices * p.a.rows)), dim3(kAdjustThreads),
         p.a.tokens != nullptr ? kSlice * sizeof(unsigned) : 0, stream, true, p);
  return check_launch("cb_adjust_logits");
}

template <typename T>
int adjust_of(const AdjustPlan& p, cudaStream_t stream) {
  return run_adjust<T, 1>(p, stream);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

int cb_adjust_logits(const cb_adjust_args* args, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_adjust_logits: null arguments");
  AdjustPlan p = {};
  p.a = *args;
  cb_adjust_args& a = p.a;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_adjust_logits: logits must be float32, bfloat16 or float16");
  CB_REQUIRE(a.rows >= 0 && a.vocab >= 0 && a.vocab < (1LL << 31) && a.rows < (1LL << 31),
             "cb_adjust_logits: %lld rows of %lld", a.rows, a.vocab);
  CB_REQUIRE(a.history >= 0 && a.history < (1LL << 31) && a.biases >= 0 && a.biases <= kMaxBiases,
             "cb_adjust_logits: a history of %lld tokens, %lld biases (at most %d)", a.history, a.biases, kMaxBiases);
  if (a.rows == 0 || a.vocab == 0) return CB_OK;
  CB_REQUIRE(a.logits != nullptr && a.out != nullptr, "cb_adjust_logits: a null pointer");
  const int item = a.dtype == CB_F32 ? 4 : 2;
  CB_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % item == 0 && reinterpret_cast<uintptr_t>(a.out) % item == 0,
             "cb_adjust_logits: logits and out must be aligned to their type");
  CB_REQUIRE(a.tokens == nullptr || a.token_dtype == CB_I32 || a.token_dtype == CB_I64,
             "cb_adjust_logits: tokens must be int32 or int64");
  CB_REQUIRE(a.tokens != nullptr || a.history == 0, "cb_adjust_logits: a history without tokens");
  CB_REQUIRE(a.biases == 0 || (a.bias != nullptr && a.bias_tokens != nullptr &&
                               (a.bias_token_dtype == CB_I32 || a.bias_token_dtype == CB_I64)),
             "cb_adjust_logits: biases need values and int32 or int64 tokens");
  if (a.history == 0) a.tokens = nullptr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == CB_F32) return adjust_of<float>(p, s);
  if (a.dtype == CB_BF16) return adjust_of<__nv_bfloat16>(p, s);
  return adjust_of<__half>(p, s);
}

}  // extern "C"
