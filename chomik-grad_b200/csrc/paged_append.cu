// Quantising writes into the paged KV cache: cb_paged_append.
//
// For a page and head, with a = max |x| over its new finite rows and s the
// scale that the page's older rows were written with (0 without any):
//   s' = max(s, a * fl(1 / top)),  q = rne(x * (1 / s')),
//   and where s' > s the older rows become rne(q * (s * (1 / s'))).
// One block per (page that the call touches, head, K or V): the largest value
// is a reduction over the block, so no scale is shared between blocks and no
// atomics are needed.  What bounds it: the rows are read once and a quarter or
// half of their bytes written (8 prompts of 2048 tokens, 8 kv heads of 128,
// bfloat16 to e4m3: 101 MB in 19.9 us, 5.1 TB/s, 78% of the measured copy, with
// 78% of the issue slots taken; one token of 32 sequences 3.8 us).  The rows stay
// in registers between the two passes (the largest value, then the codes) up to
// 8192 elements, which is a page of 64 tokens and a head of 128; beyond that they
// are read again from L2.
// The codes take few instructions: without infinities and NaN no clamp is
// needed (|x| * (1 / s') rounds to at most top), and int8 rounds by adding
// 1.5 * 2^23, whose low byte is then the code.
#include "paged.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;
constexpr int kKept = 4;                          // 8-element vectors a thread keeps
constexpr float kTiny = 7.7037197775489434e-34f;  // 2^-110
constexpr uint32_t kFinite = 0x7f7fffffu;         // bits of the largest finite float32

// Eight neighbouring elements as they are in memory.
template <int DT>
struct Vector {
  uint32_t w[DT == CB_F32 ? 8 : 4];
};

template <int DT>
__device__ __forceinline__ Vector<DT> load8(const void* base, long long at, bool wide) {
  Vector<DT> v;
  if (DT == CB_F32) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
    if (wide) {
      const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4);
      v.w[0] = a.x; v.w[1] = a.y; v.w[2] = a.z; v.w[3] = a.w;
      v.w[4 % (sizeof(v.w) / 4)] = b.x; v.w[5 % (sizeof(v.w) / 4)] = b.y;
      v.w[6 % (sizeof(v.w) / 4)] = b.z; v.w[7 % (sizeof(v.w) / 4)] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(v.w) / 4); ++i) v.w[i] = p[i];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (wide) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      v.w[0] = a.x; v.w[1] = a.y; v.w[2] = a.z; v.w[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
  }
  return v;
}

template <int DT>
__device__ __forceinline__ float element(const Vector<DT>& v, int i) {
  if (DT == CB_F32) return __uint_as_float(v.w[i]);
  const uint32_t h = i % 2 ? v.w[i / 2] >> 16 : v.w[i / 2] & 0xffffu;
  return DT == CB_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
}

// Running maximum of |x| as bits, whose order is that of the numbers, with
// infinities and NaN above all; 16-bit types: of the two halves of the words.
template <int DT>
__device__ __forceinline__ uint32_t max_bits(uint32_t most, const Vector<DT>& v) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(v.w) / 4); ++i)
    most = DT == CB_F32 ? max(most, v.w[i] & 0x7fffffffu) : __vmaxu2(most, v.w[i] & 0x7fff7fffu);
  return most;
}
template <int DT>
__device__ __forceinline__ uint32_t float_bits(uint32_t most) {
  if (DT == CB_F32) return most;
  const uint32_t h = max(most & 0xffffu, most >> 16);
  return DT == CB_BF16 ? h << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(h))));
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

// Four codes of finite numbers of at most `top` times the scale (not zero).
template <int STORAGE>
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d, float inverse) {
  if (STORAGE == CB_I8) {
    const float round = 12582912.0f;
    const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(a, inverse), round));
    const uint32_t y = __float_as_uint(__fadd_rn(__fmul_rn(b, inverse), round));
    const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(c, inverse), round));
    const uint32_t w = __float_as_uint(__fadd_rn(__fmul_rn(d, inverse), round));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inverse, b * inverse), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inverse, d * inverse), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

template <int STORAGE>
__device__ __forceinline__ float decode(uint32_t byte) {
  if (STORAGE == CB_I8) return static_cast<float>(static_cast<int8_t>(byte));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();  // shared may still be read
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = max(v, shared[w]);
  return v;
}

template <int DT, int STORAGE>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ cb_paged_append_args a, bool wide) {
  __shared__ uint32_t shared[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const cb_paged_cache& c = a.cache;
  const bool is_v = (blockIdx.x & 1) != 0;
  const int head = static_cast<int>(blockIdx.x >> 1), b = static_cast<int>(blockIdx.z);
  PagedRow row;
  if (!paged_row(c, a.sequences, a.counts, a.tokens, b, a.error_flag, &row)) return;
  const int start = row.length - row.count;
  const long long column = start / c.page + static_cast<long long>(blockIdx.y);
  if (row.count == 0 || column * c.page >= row.length) return;
  const int first = static_cast<int>(column) * c.page;
  const int page = row.table[column];
  if (page < 0 || page >= c.pages) {
    raise_flag(a.error_flag, CB_FLAG_BOOK);
    return;
  }
  const int older = max(start - first, 0);                   // rows that earlier calls wrote
  const int rows = min(row.length - first, c.page) - older;  // rows of this call
  const long long* strides = is_v ? a.v_strides : a.k_strides;
  const void* x = is_v ? a.v : a.k;
  const long long base = b * strides[0] + (first + older - start) * strides[1] + head * strides[2];
  const long long step = strides[1];
  const long long tile = (static_cast<long long>(page) * c.kv_heads + head) * c.page * c.head_size;
  uint8_t* q = static_cast<uint8_t*>(is_v ? c.v_pages : c.k_pages) + tile;
  float* scale = (is_v ? c.v_scale : c.k_scale) + static_cast<long long>(page) * c.kv_heads + head;
  const float before = older > 0 ? *scale : 0.0f;
  // vector i: row i / per_row (per_row is a power of two: head_size is 32, 64 or 128)
  const int shift = 31 - __clz(c.head_size / 8), mask = c.head_size / 8 - 1, vectors = rows << shift;
  auto load = [&](int i) { return load8<DT>(x, base + (i >> shift) * step + (i & mask) * 8, wide); };

  Vector<DT> kept[kKept];
  uint32_t most = 0;
#pragma unroll
  for (int n = 0; n < kKept; ++n) {
    const int i = n * kThreads + threadIdx.x;
    if (i < vectors) kept[n] = load(i);
  }
#pragma unroll
  for (int n = 0; n < kKept; ++n)
    if (n * kThreads + static_cast<int>(threadIdx.x) < vectors) most = max_bits<DT>(most, kept[n]);
  for (int i = kKept * kThreads + threadIdx.x; i < vectors; i += kThreads) most = max_bits<DT>(most, load(i));
  most = block_max(float_bits<DT>(most), shared);
  const bool finite = most <= kFinite;
  if (!finite) {  // once more, over the finite numbers
    most = 0;
    for (int i = threadIdx.x; i < vectors; i += kThreads) {
      const Vector<DT> v = load(i);
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = __float_as_uint(element<DT>(v, j)) & 0x7fffffffu;
        if (m <= kFinite) most = max(most, m);
      }
    }
    most = block_max(most, shared);
  }
  float grown = __uint_as_float(most) * (STORAGE == CB_I8 ? 1.0f / 127.0f : 1.0f / 448.0f);
  if (grown < kTiny) grown = 0.0f;
  const float after = fmaxf(before, grown);
  const float inverse = after == 0.0f ? 0.0f : 1.0f / after;

  uint8_t* out = q + older * c.head_size;
  if (finite && after > 0.0f) {
    auto store = [&](int i, const Vector<DT>& v) {
      *reinterpret_cast<uint2*>(out + i * 8) =
          make_uint2(quantise4<STORAGE>(element<DT>(v, 0), element<DT>(v, 1), element<DT>(v, 2), element<DT>(v, 3), inverse),
                     quantise4<STORAGE>(element<DT>(v, 4), element<DT>(v, 5), element<DT>(v, 6), element<DT>(v, 7), inverse));
    };
#pragma unroll
    for (int n = 0; n < kKept; ++n) {
      const int i = n * kThreads + threadIdx.x;
      if (i < vectors) store(i, kept[n]);
    }
    for (int i = kKept * kThreads + threadIdx.x; i < vectors; i += kThreads) store(i, load(i));
  } else {
    for (int i = threadIdx.x; i < vectors; i += kThreads) {
      const Vector<DT> v = load(i);
      uint2 codes = make_uint2(0u, 0u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        codes.x |= quantise<STORAGE>(element<DT>(v, j), inverse) << (8 * j);
        codes.y |= quantise<STORAGE>(element<DT>(v, 4 + j), inverse) << (8 * j);
      }
      *reinterpret_cast<uint2*>(out + i * 8) = codes;
    }
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
  if (a.cache.storage == CB_I8) launch(append_kernel<DT, CB_I8>, grid, dim3(kThreads), 0, stream, true, a, wide);
  else launch(append_kernel<DT, CB_E4M3>, grid, dim3(kThreads), 0, stream, true, a, wide);
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
