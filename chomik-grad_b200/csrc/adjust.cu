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
// and 1/8 of the mask), and few tokens have more than the mask.  A block takes a
// slice of one row's vocabulary, with a word for each of its tokens in shared memory,
// where the history (read by every slice of the row, from L2) and the biases are
// counted; it copies the slice under the mask; then the tokens of the history and of
// the biases, each by the first thread that claims it, are adjusted where they now are.
// (With every token adjusted in the copy, 47 instructions a token, 64 rows of 128256
// took 41 us.)  They now take 22; 80 rows of 32003 with a mask alone 4; one of 32000
// 4.3, a launch and a chain of loads.  A token's biases are summed by the thread of its first entry, in the
// list's order (no float atomics: equal inputs give equal bits).
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kAdjustThreads = 512;
constexpr int kMaxBiases = 1023;
constexpr int kWideFrom = 6;  // slices of 4096 tokens to an SM
constexpr int kHeld = 8;  // tokens of the history that a thread holds in registers
// A token's word: how often it was made, the number of its sum of biases (0: none),
// whether it is anywhere in the history, and whether a thread has claimed it.
constexpr unsigned kCount = 0xfffffu, kBias = 0x3ffu, kClaimed = 0x40000000u, kSeen = 0x80000000u;
constexpr int kBiasAt = 20;

struct AdjustPlan {
  cb_adjust_args a;
  int slices;         // of a row
  int has_history;    // tokens, or lengths to be checked
  int shared_lead;    // logits and out lie alike to 16 bytes in every row: wide accesses
};

struct Penalty {
  float repetition, frequency, presence;
};

__device__ __forceinline__ float adjusted(float x, unsigned word, const Penalty& p, const float* sums) {
  const unsigned made = word & kCount, bias = word >> kBiasAt & kBias;
  if ((word & (kSeen | kCount)) != 0) x = x > 0.0f ? x / p.repetition : x * p.repetition;
  if (made != 0) x -= fmaf(p.frequency, static_cast<float>(made), p.presence);
  if (bias != 0) x += sums[bias - 1];
  return x;
}

__device__ __forceinline__ bool is_allowed(const int* allowed, int v) {
  return allowed == nullptr || (static_cast<unsigned>(allowed[v >> 5]) >> (v & 31) & 1u) != 0;
}

// Eight neighbouring elements as they are in memory: one 16-byte access for 16-bit
// types, two for float32.  mask: those whose bit is clear become -inf.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  static constexpr int kCode = CB_F32;
  float x[8];
  __device__ __forceinline__ void set(int i, float v) { x[i] = v; }
  __device__ __forceinline__ float get(int i) const { return x[i]; }
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
  __device__ __forceinline__ void mask(unsigned bits) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (bits >> i & 1u) != 0 ? x[i] : -INFINITY;
  }
};
template <typename T, int CODE, uint32_t LOWEST>
struct EightHalves {
  static constexpr int kCode = CODE;
  uint32_t w[4];
  __device__ __forceinline__ T get(int i) const {
    const uint16_t h = static_cast<uint16_t>(w[i / 2] >> (i % 2 * 16));
    return *reinterpret_cast<const T*>(&h);
  }
  __device__ __forceinline__ void set(int i, T v) {
    const uint32_t h = *reinterpret_cast<const uint16_t*>(&v);
    w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | h << 16 : (w[i / 2] & 0xffff0000u) | h;
  }
  __device__ __forceinline__ void load(const void* p) {
    const uint4 v = *static_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void store(void* p) const {
    *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void mask(unsigned bits) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t keep = ((bits >> 2 * i & 1u) * 0xffffu) | ((bits >> (2 * i + 1) & 1u) * 0xffff0000u);
      w[i] = (w[i] & keep) | (LOWEST & ~keep);
    }
  }
};
template <>
struct Eight<__nv_bfloat16> : EightHalves<__nv_bfloat16, CB_BF16, 0xff80ff80u> {};
template <>
struct Eight<__half> : EightHalves<__half, CB_F16, 0xfc00fc00u> {};

// EIGHTS: runs of eight neighbouring tokens that a thread takes.
template <typename T, int EIGHTS>
__global__ void __launch_bounds__(kAdjustThreads) adjust_kernel(const __grid_constant__ AdjustPlan p) {
  constexpr int kSlice = kAdjustThreads * 8 * EIGHTS, kOwn = (kMaxBiases + 1) / kAdjustThreads;
  extern __shared__ __align__(16) unsigned words[];  // of the slice's tokens, where there is a history or biases
  __shared__ __align__(16) int listed[kMaxBiases + 1];   // the biases' places, -1 for those outside the slice
  __shared__ float sums[kMaxBiases + 1];
  const cb_adjust_args& a = p.a;
  const long long row = blockIdx.x / p.slices;
  const int thread = threadIdx.x;
  const bool listed_tokens = p.has_history != 0, counted = listed_tokens || a.biases > 0;
  pdl_launch_dependents();
  pdl_wait();

  const T* in = static_cast<const T*>(a.logits) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.out_ld;
  // Places are counted from the last 16-byte boundary at or before the row's
  // beginning: token = place - lead.
  const int lead = p.shared_lead ? static_cast<int>(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T)) : 0;
  const int first = static_cast<int>(blockIdx.x % p.slices) * kSlice - lead;  // token of place 0
  const int vocab = static_cast<int>(a.vocab), history = static_cast<int>(a.history);
  const int* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_ld : nullptr;

  Eight<T> x[EIGHTS];
  auto token_of = [&](int n) { return first + (n * kAdjustThreads + thread) * 8; };
  auto whole = [&](int v) { return p.shared_lead && v >= 0 && v + 8 <= vocab; };
  // entry i of a list as a place of the slice, -1 where it is not in it
  auto place_of = [&](const void* list, int dtype, int i) {
    if (dtype == CB_I32) {
      const int token = static_cast<const int*>(list)[i];
      return token >= 0 && token < vocab && token >= first && token - first < kSlice ? token - first : -1;
    }
    const long long token = static_cast<const long long*>(list)[i];
    const long long place = token - first;
    return place >= 0 && place < kSlice && token >= 0 && token < vocab ? static_cast<int>(place) : -1;
  };
#pragma unroll
  for (int n = 0; n < EIGHTS; ++n) {
    const int v = token_of(n);
    if (whole(v)) {
      x[n].load(in + v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v + i >= 0 && v + i < vocab) x[n].set(i, in[v + i]);
    }
  }
  unsigned bits[EIGHTS];  // of the mask
#pragma unroll
  for (int n = 0; n < EIGHTS; ++n) {
    const int v = token_of(n), low = max(v, 0), word = low >> 5;
    bits[n] = 0xffu;
    if (allowed != nullptr && v + 8 > 0 && v < vocab) {
      const unsigned a0 = allowed[word], a1 = word < (vocab - 1) >> 5 ? allowed[word + 1] : 0;
      bits[n] = __funnelshift_r(a0, a1, low & 31) << (low - v);
    }
  }
  Penalty penalty{a.repetition, a.frequency, a.presence};
  const char* tokens = static_cast<const char*>(a.tokens) + row * a.token_ld * (a.token_dtype == CB_I64 ? 8 : 4);
  const char* ids = static_cast<const char*>(a.bias_tokens) + row * a.bias_token_ld * (a.bias_token_dtype == CB_I64 ? 8 : 4);
  int length = 0, prompt = 0, held[kHeld], own[kOwn];  // places
  float bias_of[kOwn];
  if (counted) {
    if (listed_tokens) {
#pragma unroll
      for (int n = 0; n < kHeld; ++n) {
        const int i = n * kAdjustThreads + thread;
        held[n] = i < history ? place_of(tokens, a.token_dtype, i) : -1;
      }
      length = a.lengths != nullptr ? a.lengths[row] : history;
      prompt = a.prompts != nullptr ? a.prompts[row] : 0;
      if (a.repetitions != nullptr) penalty.repetition = a.repetitions[row];
      if (a.frequencies != nullptr) penalty.frequency = a.frequencies[row];
      if (a.presences != nullptr) penalty.presence = a.presences[row];
    }
    const int biases = static_cast<int>(a.biases);
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
      const int i = n * kAdjustThreads + thread;
      own[n] = i < biases ? place_of(ids, a.bias_token_dtype, i) : -1;
      bias_of[n] = i < biases ? a.bias[row * a.bias_ld + i] : 0.0f;
      if (i < (biases + 3) / 4 * 4) listed[i] = own[n];
    }
    for (int i = thread; i < kSlice / 4; i += kAdjustThreads)
      reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    if (length < 0 || length > history || prompt < 0 || prompt > length) {
      raise_flag(a.error_flag, CB_FLAG_HISTORY);
      length = min(max(length, 0), history);
      prompt = min(max(prompt, 0), length);
    }
    __syncthreads();
    auto count = [&](int i, int place) {
      if (place >= 0 && i < length) {
        if (i >= prompt) atomicAdd(words + place, 1u);
        else atomicOr(words + place, kSeen);
      }
    };
    if (listed_tokens) {
#pragma unroll
      for (int n = 0; n < kHeld; ++n) count(n * kAdjustThreads + thread, held[n]);
      for (int i = kHeld * kAdjustThreads + thread; i < length; i += kAdjustThreads)
        count(i, place_of(tokens, a.token_dtype, i));
    }
    if (a.biases > 0) {
      const float* bias = a.bias + row * a.bias_ld;
#pragma unroll
      for (int n = 0; n < kOwn; ++n) {
        const int mine = n * kAdjustThreads + thread, v = own[n];
        if (v < 0) continue;
        bool earlier = false;
        float sum = 0.0f;
        for (int i = 0; i < biases; i += 4) {  // (the list is padded with -1)
          const int4 four = *reinterpret_cast<const int4*>(listed + i);
          if (four.x != v && four.y != v && four.z != v && four.w != v) continue;
          const int same[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (same[k] != v) continue;
            earlier = earlier || i + k < mine;
            sum = i + k == mine ? bias_of[n] : sum + bias[i + k];
          }
        }
        if (earlier) continue;
        sums[mine] = sum;
        atomicOr(words + v, static_cast<unsigned>(mine + 1) << kBiasAt);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < EIGHTS; ++n) {
    const int v = token_of(n);
    if (v + 8 <= 0 || v >= vocab) continue;
    x[n].mask(bits[n]);
    if (whole(v)) {
      x[n].store(out + v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v + i >= 0 && v + i < vocab) out[v + i] = x[n].get(i);
    }
  }
  if (!counted) return;
  __syncthreads();  // the slice is copied and every word is complete
  // `places` (-1: none): claimed, then loaded, then adjusted, so that the loads of all are
  // in flight together; a masked token stays -inf
  auto adjust = [&](auto& places) {
    constexpr int kPlaces = sizeof(places) / sizeof(places[0]);
    unsigned word[kPlaces];
    float was[kPlaces];
    bool fine[kPlaces];
#pragma unroll
    for (int n = 0; n < kPlaces; ++n) word[n] = places[n] >= 0 ? atomicOr(words + places[n], kClaimed) : kClaimed;
#pragma unroll
    for (int n = 0; n < kPlaces; ++n) {
      was[n] = 0.0f;
      fine[n] = (word[n] & kClaimed) == 0;
      if (fine[n]) {
        was[n] = load_as_f32(out, places[n] + first, Eight<T>::kCode);
        fine[n] = is_allowed(allowed, places[n] + first);
      }
    }
#pragma unroll
    for (int n = 0; n < kPlaces; ++n)
      if (fine[n]) store_from_f32(out, places[n] + first, Eight<T>::kCode, adjusted(was[n], word[n], penalty, sums));
  };
  if (listed_tokens) {
#pragma unroll
    for (int n = 0; n < kHeld; ++n)
      if (n * kAdjustThreads + thread >= length) held[n] = -1;
    adjust(held);
    for (int from = kHeld * kAdjustThreads; from < length; from += kHeld * kAdjustThreads) {
#pragma unroll
      for (int n = 0; n < kHeld; ++n) {
        const int i = from + n * kAdjustThreads + thread;
        held[n] = i < length ? place_of(tokens, a.token_dtype, i) : -1;
      }
      adjust(held);
    }
  }
  if (a.biases > 0) adjust(own);
}

template <typename T, int EIGHTS>
int run_adjust(AdjustPlan p, cudaStream_t stream) {
  constexpr int kSlice = kAdjustThreads * 8 * EIGHTS;
  const long long item = sizeof(T);
  const uintptr_t in = reinterpret_cast<uintptr_t>(p.a.logits), out = reinterpret_cast<uintptr_t>(p.a.out);
  p.shared_lead = (in - out) % 16 == 0 && (p.a.rows == 1 || (p.a.ld - p.a.out_ld) * item % 16 == 0);
  const long long slices = (p.a.vocab + 7 + kSlice - 1) / kSlice;
  CB_REQUIRE(slices * p.a.rows < (1LL << 31), "cb_adjust_logits: %lld rows of %lld", p.a.rows, p.a.vocab);
  p.slices = static_cast<int>(slices);
  const size_t words = p.has_history || p.a.biases > 0 ? kSlice * sizeof(unsigned) : 0;
  if (words > 40 * 1024) {
    static thread_local int device = -1;
    int now = 0;
    cudaGetDevice(&now);
    if (now != device) {
      const cudaError_t e = cudaFuncSetAttribute(adjust_kernel<T, EIGHTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(words));
      CB_REQUIRE(e == cudaSuccess, "cb_adjust_logits: %s", cudaGetErrorString(e));
      device = now;
    }
  }
  launch(adjust_kernel<T, EIGHTS>, dim3(static_cast<unsigned>(slices * p.a.rows)), dim3(kAdjustThreads), words, stream,
         true, p);
  return check_launch("cb_adjust_logits");
}

template <typename T>
int adjust_of(const AdjustPlan& p, cudaStream_t stream) {
  // Slices of 4096 tokens fill the GPU at few rows (1 of 32000 with a history of 2048:
  // 4.6 us, of 16384 4.6 as well, on fewer SMs); more rows share the work of a slice (its
  // history, biases and waits) between more tokens (64 rows of 128256, histories of 4000:
  // 24 us with slices of 16384, 33 of 8192, 50 of 4096).
  const long long blocks = p.a.rows * ((p.a.vocab + 4095) / 4096);
  if (!p.has_history && p.a.biases == 0) return run_adjust<T, 1>(p, stream);
  if (blocks > kWideFrom * sm_count()) return run_adjust<T, 4>(p, stream);
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
  CB_REQUIRE(a.rows >= 0 && a.vocab >= 0 && a.vocab < (1LL << 30) && a.rows < (1LL << 31),
             "cb_adjust_logits: %lld rows of %lld", a.rows, a.vocab);
  CB_REQUIRE(a.history >= 0 && a.history <= kCount && a.biases >= 0 && a.biases <= kMaxBiases,
             "cb_adjust_logits: a history of %lld tokens, %lld biases (at most %d)", a.history, a.biases, kMaxBiases);
  if (a.rows == 0 || a.vocab == 0) return CB_OK;
  CB_REQUIRE(a.logits != nullptr && a.out != nullptr, "cb_adjust_logits: a null pointer");
  const int item = a.dtype == CB_F32 ? 4 : 2;
  CB_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % item == 0 && reinterpret_cast<uintptr_t>(a.out) % item == 0,
             "cb_adjust_logits: logits and out must be aligned to their type");
  CB_REQUIRE(a.rows == 1 || a.out_ld >= a.vocab || -a.out_ld >= a.vocab,
             "cb_adjust_logits: rows of %lld tokens, %lld apart, share memory", a.vocab, a.out_ld);
  CB_REQUIRE(a.tokens == nullptr || a.token_dtype == CB_I32 || a.token_dtype == CB_I64,
             "cb_adjust_logits: tokens must be int32 or int64");
  CB_REQUIRE(a.tokens != nullptr || a.history == 0, "cb_adjust_logits: a history without tokens");
  CB_REQUIRE(a.biases == 0 || (a.bias != nullptr && a.bias_tokens != nullptr &&
                               (a.bias_token_dtype == CB_I32 || a.bias_token_dtype == CB_I64)),
             "cb_adjust_logits: biases need values and int32 or int64 tokens");
  p.has_history = a.history > 0 || a.lengths != nullptr || a.prompts != nullptr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == CB_F32) return adjust_of<float>(p, s);
  if (a.dtype == CB_BF16) return adjust_of<__nv_bfloat16>(p, s);
  return adjust_of<__half>(p, s);
}

}  // extern "C"
