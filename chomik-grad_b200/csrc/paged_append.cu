// Quantising writes into the paged KV cache: cb_paged_append.
//
// For a page and head, with a = max |x| over its new finite rows and s the
// scale that the page's older rows were written with (0 without any):
//   s' = max(s, a * fl(1 / top)),  q = rne(x * (1 / s')),
//   and where s' > s the older rows become rne(q * (s * (1 / s'))).
// One block per (page that the call touches, head, K or V): the largest value
// is a reduction over the block, so no scale is shared between blocks and no
// atomics are needed.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;
constexpr float kTiny = 7.7037197775489434e-34f;  // 2^-110

template <int DT>
__device__ __forceinline__ void load8(const void* base, long long at, bool wide, float* x) {
  if (DT == CB_F32) {
    const float* p = static_cast<const float*>(base) + at;
    if (wide) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    uint16_t h[8];
    if (wide) {
      *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = DT == CB_BF16 ? bf16_bits_to_f32(h[i]) : __half2float(__ushort_as_half(h[i]));
  }
}

template <int STORAGE>
__device__ __forceinline__ uint32_t quantise(float x, float inverse) {
  float y = inverse == 0.0f ? 0.0f : x * inverse;
  if (STORAGE == CB_I8) {
    const int q = __float2int_rn(y);  // NaN gives 0, infinities saturate
    return static_cast<uint32_t>(min(max(q, -127), 127)) & 0xffu;
  }
  if (y != y) y = 0.0f;
  return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

template <int STORAGE>
__device__ __forceinline__ float decode(uint32_t byte) {
  if (STORAGE == CB_I8) return static_cast<float>(static_cast<int8_t>(byte));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

template <int DT, int STORAGE>
__global__ void __launch_bounds__(kThreads) append_kernel(cb_paged_append_args a, bool wide) {
  const cb_paged_cache& c = a.cache;
  const bool is_v = (blockIdx.x & 1) != 0;
  const int head = static_cast<int>(blockIdx.x >> 1), b = static_cast<int>(blockIdx.z);
  PagedRow row;
  if (!paged_row(c, a.sequences, a.counts, a.tokens, b, a.error_flag, &row)) return;
  const int start = row.length - row.count;
  const int column = start / c.page + static_cast<int>(blockIdx.y);
  const int first = column * c.page;
  if (row.count == 0 || first >= row.length) return;
  const int page = row.table[column];
  if (page < 0 || page >= c.pages) {
    raise_flag(a.error_flag, CB_FLAG_BOOK);
    return;
  }
  const int older = max(start - first, 0);                       // rows that earlier calls wrote
  const int rows = min(row.length - first, c.page) - older;      // rows of this call
  const long long* strides = is_v ? a.v_strides : a.k_strides;
  const void* x = is_v ? a.v : a.k;
  const long long base = b * strides[0] + (first + older - start) * strides[1] + head * strides[2];
  const long long tile = (static_cast<long long>(page) * c.kv_heads + head) * c.page * c.head_size;
  uint8_t* q = static_cast<uint8_t*>(is_v ? c.v_pages : c.k_pages) + tile;
  float* scale = (is_v ? c.v_scale : c.k_scale) + static_cast<long long>(page) * c.kv_heads + head;
  const float before = older > 0 ? *scale : 0.0f;
  const int vectors = rows * c.head_size / 8, per_row = c.head_size / 8;

  float largest = 0.0f;
  for (int i = threadIdx.x; i < vectors; i += kThreads) {
    float v[8];
    load8<DT>(x, base + (i / per_row) * strides[1] + (i % per_row) * 8, wide, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float m = fabsf(v[j]);
      if (m <= 3.4028234663852886e38f) largest = fmaxf(largest, m);
    }
  }
  __shared__ float shared[kThreads / 32];
  largest = warp_max(largest);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = largest;
  __syncthreads();
  largest = shared[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) largest = fmaxf(largest, shared[w]);
  float grown = largest * (STORAGE == CB_I8 ? 1.0f / 127.0f : 1.0f / 448.0f);
  if (grown < kTiny) grown = 0.0f;
  const float after = fmaxf(before, grown);
  const float inverse = after == 0.0f ? 0.0f : 1.0f / after;

  for (int i = threadIdx.x; i < vectors; i += kThreads) {
    float v[8];
    load8<DT>(x, base + (i / per_row) * strides[1] + (i % per_row) * 8, wide, v);
    uint2 out = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out.x |= quantise<STORAGE>(v[j], inverse) << (8 * j);
      out.y |= quantise<STORAGE>(v[4 + j], inverse) << (8 * j);
    }
    *reinterpret_cast<uint2*>(q + older * c.head_size + i * 8) = out;
  }
  if (after > before && older > 0) {
    const float ratio = before * inverse;
    for (int i = threadIdx.x; i < older * c.head_size / 4; i += kThreads) {
      uint32_t* p = reinterpret_cast<uint32_t*>(q) + i;
      const uint32_t was = *p;
      uint32_t now = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) now |= quantise<STORAGE>(decode<STORAGE>((was >> (8 * j)) & 0xffu), ratio) << (8 * j);
      *p = now;
    }
  }
  if (threadIdx.x == 0) *scale = after;
}

template <int DT>
int launch_append(const cb_paged_append_args& a, bool wide, dim3 grid, cudaStream_t stream) {
  if (a.cache.storage == CB_I8) append_kernel<DT, CB_I8><<<grid, kThreads, 0, stream>>>(a, wide);
  else append_kernel<DT, CB_E4M3><<<grid, kThreads, 0, stream>>>(a, wide);
  return check_launch("cb_paged_append");
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_paged_append(const cb_paged_append_args* args, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_paged_append: null arguments");
  const cb_paged_append_args& a = *args;
  const int status = paged_cache_check(a.cache, "cb_paged_append");
  if (status != CB_OK) return status;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_paged_append: k and v must be float32, bfloat16 or float16");
  CB_REQUIRE(a.batch >= 0 && a.batch <= 65535 && a.tokens >= 0, "cb_paged_append: %lld sequences of %lld tokens",
             a.batch, a.tokens);
  if (a.batch == 0 || a.tokens == 0) return CB_OK;
  CB_REQUIRE(a.k != nullptr && a.v != nullptr, "cb_paged_append: a null pointer");
  const long long touched = (a.tokens + a.cache.page - 2) / a.cache.page + 1;
  CB_REQUIRE(touched <= 65535, "cb_paged_append: %lld tokens are too many for one call", a.tokens);
  const int item = a.dtype == CB_F32 ? 4 : 2;
  bool wide = reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  for (int i = 0; i < 3; ++i) wide = wide && a.k_strides[i] * item % 16 == 0 && a.v_strides[i] * item % 16 == 0;
  const dim3 grid(2 * a.cache.kv_heads, static_cast<unsigned>(touched), static_cast<unsigned>(a.batch));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == CB_F32) return launch_append<CB_F32>(a, wide, grid, s);
  if (a.dtype == CB_BF16) return launch_append<CB_BF16>(a, wide, grid, s);
  return launch_append<CB_F16>(a, wide, grid, s);
}
