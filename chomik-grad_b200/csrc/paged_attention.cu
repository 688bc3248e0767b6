// Attention over the paged 8-bit KV cache: cb_paged_attention.
//
// For the query row of token t of the last n of a slot with `length` keys,
// head h of kv head g = h / (heads / kv_heads):
//   s_j = scale * ks[page(j), g] * sum_d q_d kq[j, d],  j <= length - n + t
//   out = sum_j exp(s_j - m) vs[page(j), g] vq[j, :] / sum_j exp(s_j - m)
// in one pass over the keys, with the running maximum m and sum.
//
// One block per (sequence, token, head); each warp takes every fourth key, its
// lanes hold head_size / 32 neighbouring elements each, and the warps' partial
// results are joined in shared memory.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

template <int STORAGE>
__device__ __forceinline__ float decode(uint8_t byte) {
  if (STORAGE == CB_I8) return static_cast<float>(static_cast<int8_t>(byte));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3)));
}

template <int STORAGE>
__global__ void __launch_bounds__(kThreads) attention_kernel(cb_paged_attention_args a) {
  const cb_paged_cache& c = a.cache;
  const int h = static_cast<int>(blockIdx.x), t = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const int g = h / static_cast<int>(a.heads / c.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = c.head_size / 32;
  PagedRow row;
  const bool ok = paged_row(c, a.sequences, a.counts, a.tokens, b, a.error_flag, &row);
  const int keys = ok && t < row.count ? row.length - row.count + t + 1 : 0;
  float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  for (int i = 0; i < per; ++i)
    q[i] = load_as_f32(a.q, b * a.q_strides[0] + t * a.q_strides[1] + h * a.q_strides[2] + lane * per + i, a.dtype);
  for (int j = warp; j < keys; j += kWarps) {
    const int page = row.table[j / c.page];
    if (page < 0 || page >= c.pages) {
      raise_flag(a.error_flag, CB_FLAG_BOOK);
      continue;
    }
    const long long block = static_cast<long long>(page) * c.kv_heads + g;
    const long long at = (block * c.page + j % c.page) * c.head_size + lane * per;
    float s = 0.0f;
    for (int i = 0; i < per; ++i) s += q[i] * decode<STORAGE>(static_cast<const uint8_t*>(c.k_pages)[at + i]);
    s = warp_sum(s) * (c.k_scale[block] * a.scale * 1.4426950408889634f);
    const float top = fmaxf(m, s), keep = exp2f(m - top), p = exp2f(s - top);
    int exponent;  // of the value scale, which may make up for a weight below float32's range
    const float fraction = frexpf(c.v_scale[block], &exponent);
    const float weight = exp2f(s - top + exponent) * fraction;
    l = l * keep + p;
    for (int i = 0; i < per; ++i)
      o[i] = o[i] * keep + weight * decode<STORAGE>(static_cast<const uint8_t*>(c.v_pages)[at + i]);
    m = top;
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][128];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int i = 0; i < per; ++i) so[warp][lane * per + i] = o[i];
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < c.head_size) {
    float top = -INFINITY, sum = 0.0f, v = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kWarps && keys > 0; ++w) {
      const float f = sm[w] == -INFINITY ? 0.0f : exp2f(sm[w] - top);
      sum += f * sl[w];
      v += f * so[w][threadIdx.x];
    }
    const long long at = ((b * a.tokens + t) * a.heads + h) * c.head_size + threadIdx.x;
    store_from_f32(a.out, at, a.dtype, sum > 0.0f || sum != sum ? v / sum : 0.0f);
  }
}

int attention_check(const cb_paged_attention_args& a) {
  const int status = paged_cache_check(a.cache, "cb_paged_attention");
  if (status != CB_OK) return status;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_paged_attention: q must be float32, bfloat16 or float16");
  CB_REQUIRE(a.heads >= 1 && a.heads % a.cache.kv_heads == 0, "cb_paged_attention: %lld heads for %d kv heads",
             a.heads, a.cache.kv_heads);
  CB_REQUIRE(a.batch >= 0 && a.batch <= 65535 && a.tokens >= 0 && a.tokens <= 65535,
             "cb_paged_attention: %lld sequences of %lld tokens", a.batch, a.tokens);
  return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_paged_attention_scratch(const cb_paged_attention_args* args) {
  (void)args;
  return 0;
}

int cb_paged_attention(const cb_paged_attention_args* args, void* scratch, cb_stream_t stream) {
  (void)scratch;
  CB_REQUIRE(args != nullptr, "cb_paged_attention: null arguments");
  const cb_paged_attention_args& a = *args;
  const int status = attention_check(a);
  if (status != CB_OK) return status;
  if (a.batch == 0 || a.tokens == 0) return CB_OK;
  CB_REQUIRE(a.q != nullptr && a.out != nullptr, "cb_paged_attention: a null pointer");
  const dim3 grid(static_cast<unsigned>(a.heads), static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.batch));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.cache.storage == CB_I8) attention_kernel<CB_I8><<<grid, kThreads, 0, s>>>(a);
  else attention_kernel<CB_E4M3><<<grid, kThreads, 0, s>>>(a);
  return check_launch("cb_paged_attention");
}

}  // extern "C"
