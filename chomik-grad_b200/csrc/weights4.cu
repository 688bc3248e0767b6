// Products with 4-bit weights and group scales: cb_weights4_linear, and what makes
// and unmakes such weights (cb_weights4_quantise, _pack, _dequantise).
//
//   y[m, n] = sum over groups g of s[n, g] * sum_{k in g} q[n, k] x[m, k],  q in [-8, 7]
//
// What bounds it: the weights are read once, half a byte each and 2 bytes for a
// group's scale, 2 flops a weight and row.  At the measured 6.46 TB/s an SM gets 23
// bytes a clock, 46 weights: with scalar multiply-adds that would be 46 conversions
// and as many products for each row, so the products go to the tensor cores
// (m16n8k16, float32 sums) with the weights as the 16-row operand: up to 8 columns
// cost the same.  The codes are exact in fp16 and bfloat16, so x stays in its own
// type, and a group's scale multiplies the group's float32 sum, which has to be within
// float32 before that.  float32 x is split into three bfloat16 parts that are columns of
// their own (24 bits; of numbers below 2^-110 what is above 2^-133), so 2 rows of it cost
// what one does.
//
// Layout.  The operand's order of k is free as long as x has the same, so weights
// are kept as a lane reads them: a block of 16 outputs x 64 inputs is 512 bytes, 16
// for each lane (row g = lane / 4 and g + 8, c = lane % 4), one word for each
// product: word s of lane (g, c) holds inputs k = 32 (s / 2) + 8 c + 4 (s % 2) + 0 .. 3
// of both rows.  Lane (g, c) so needs x[g][32 h + 8 c + 0 .. 7], 16 neighbouring bytes,
// which come straight from L1: no staging, no barrier before the products.  Measured:
// 16 rows by 4096 x 128256, 77 us (3.6 TB/s: 16 warps an SM do not cover the loads of
// x and the conversions), one row 55 (5.0 TB/s); one row by 4096 x 14336 8.2, by 2048 x
// 2048 2.2, a launch and one chain of loads, products and sums.  Above 16 rows a block has
// one tile and loads all of them from L1 for it, and above 32 the weights are read and
// converted again: 24, 32, 64 and 80 rows by 4096 x 128256 take 134, 179, 354 and 498 us.  Code
// q + 8 of pair i (row g, inputs 0 and 1; row g + 8, the same; row g, inputs 2 and
// 3; row g + 8) is nibbles i and i + 4: one logic instruction makes two operands of
// them (see halves_of).
#include <type_traits>

#include "common.cuh"

namespace cb {
namespace {

constexpr int kBlockBytes = 512;   // 16 outputs x 64 inputs
constexpr int kColumnTiles = 4;    // most of 8 columns that a launch's block takes

__host__ __device__ constexpr long long tiles_of(long long outputs) { return (outputs + 15) / 16; }
__host__ __device__ constexpr long long chunks_of(long long inputs) { return (inputs + 63) / 64; }
// Scales of a tile: by chunk (two chunks, for groups of 128), row g, group within the chunk, rows g and g + 8.
__host__ __device__ constexpr long long tile_scales(long long inputs, int group) {
  return group == 128 ? (chunks_of(inputs) + 1) / 2 * 16 : chunks_of(inputs) * (64 / group) * 16;
}
__device__ __forceinline__ float scale_of(uint32_t bits, int dtype) {
  return dtype == CB_BF16 ? bf16_bits_to_f32(static_cast<uint16_t>(bits))
                          : __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
}

// Pair i of a word as two numbers of the products' type.  bfloat16: the code under
// the exponent of 128 is 128 + code; fp16: under that of 1024, where the next
// nibble is in reach too, as 1024 + 16 * code.  (The method: Kim, Henry, Fahim and Awadalla,
// "Who Says Elephants Can't Run", 2022.)
template <bool HALF>
__device__ __forceinline__ void halves_of(uint32_t w, uint32_t* a) {
  if (HALF) {
    const __half2 low = __half2half2(__ushort_as_half(0x6408));                  // 1032
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00)), high = __half2half2(__ushort_as_half(0xd480));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = i ? w >> 8 : w;
      uint32_t x, y;
      asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x) : "r"(v));  // (v & mask) | bits
      asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(y) : "r"(v));
      __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), low);
      __half2 q = __hfma2(*reinterpret_cast<__half2*>(&y), sixteenth, high);     // (1024 + 16 code) / 16 - 72
      a[2 * i] = *reinterpret_cast<uint32_t*>(&p);
      a[2 * i + 1] = *reinterpret_cast<uint32_t*>(&q);
    }
  } else {
    const __nv_bfloat162 bias = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x;
      asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(x) : "r"(w >> 4 * i));
      __nv_bfloat162 p = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), bias);
      a[i] = *reinterpret_cast<uint32_t*>(&p);
    }
  }
}

template <bool HALF>
__device__ __forceinline__ void product(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (HALF) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

struct LinearPlan {
  cb_weights4 w;
  const void* x;  // 16-bit rows, 16-byte aligned
  long long ld;   // elements between them
  int rows;       // of x, of all launches' blocks
  int parts;      // rows of x that a row of y is the sum of: part p of row r is row p * (rows / parts) + r
  void* out;
  int out_dtype;
  long long out_ld;
  int per;  // rows of y that a block takes
};

// A unit of a warp: 16 outputs x 128 inputs, and their scales.
template <int GROUP>
struct Unit {
  static constexpr int kWords = GROUP == 32 ? 4 : GROUP == 64 ? 2 : 1;
  uint4 codes[2];
  uint32_t scales[kWords];
};
// WHOLE: both of its chunks are there.
template <int GROUP, bool WHOLE>
__device__ __forceinline__ void load_unit(Unit<GROUP>& u, const uint4* codes, const uint32_t* scales) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool real = WHOLE || i == 0;
    u.codes[i] = real ? __ldcs(codes + i * 32) : make_uint4(0, 0, 0, 0);
    if (GROUP == 64) u.scales[i % Unit<GROUP>::kWords] = real ? __ldcs(scales + i * 8) : 0;
    if (GROUP == 32) {
      const uint2 two = real ? __ldcs(reinterpret_cast<const uint2*>(scales) + i * 8) : make_uint2(0, 0);
      u.scales[2 * i % Unit<GROUP>::kWords] = two.x;
      u.scales[(2 * i + 1) % Unit<GROUP>::kWords] = two.y;
    }
  }
  if (GROUP == 128) u.scales[0] = __ldcs(scales);
}

// The products of TILES units with the same x.  `left`: inputs from this lane's first on
// (all of a whole unit's are there).
template <bool HALF, int GROUP, int COLUMNS, int TILES, bool WHOLE>
__device__ __forceinline__ void multiply_units(const Unit<GROUP>* u, const uint16_t* const* x, long long k, long long left,
                                               int scale_dtype, float (*total)[COLUMNS][4]) {
  float sum[TILES][COLUMNS][4];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = part * 64 + h * 32;
      uint4 b[COLUMNS];
#pragma unroll
      for (int t = 0; t < COLUMNS; ++t)
        b[t] = WHOLE || at < left ? *reinterpret_cast<const uint4*>(x[t] + k + at) : make_uint4(0, 0, 0, 0);
      const bool begins = GROUP == 32 || (h == 0 && (GROUP == 64 || part == 0));
      const bool ends = GROUP == 32 || (h == 1 && (GROUP == 64 || part == 1));
#pragma unroll
      for (int n = 0; n < TILES; ++n) {
        const uint32_t w[4] = {u[n].codes[part].x, u[n].codes[part].y, u[n].codes[part].z, u[n].codes[part].w};
        uint32_t a[4];
        halves_of<HALF>(w[2 * h], a);
#pragma unroll
        for (int t = 0; t < COLUMNS; ++t) {
          if (begins) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[n][t][i] = 0.0f;
          }
          product<HALF>(sum[n][t], a, b[t].x, b[t].y);
        }
        halves_of<HALF>(w[2 * h + 1], a);
#pragma unroll
        for (int t = 0; t < COLUMNS; ++t) product<HALF>(sum[n][t], a, b[t].z, b[t].w);
        if (ends) {
          const uint32_t both = u[n].scales[GROUP == 32 ? 2 * part + h : GROUP == 64 ? part : 0];
          const float low = scale_of(both & 0xffffu, scale_dtype), high = scale_of(both >> 16, scale_dtype);
#pragma unroll
          for (int t = 0; t < COLUMNS; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[n][t][i] = fmaf(i < 2 ? low : high, sum[n][t][i], total[n][t][i]);
        }
      }
    }
  }
}

// A block takes TILES tiles of 16 outputs and `per` rows of y.  Its WARPS warps take the
// units of the tiles in turn, the loads of the next under way, and are joined in
// shared memory, in their order.  Columns that no row of x belongs to are computed
// like row `first` and not stored.
template <bool HALF, int GROUP, int COLUMNS, int TILES, int WARPS, int RESIDENT>
__global__ void __launch_bounds__(32 * WARPS, RESIDENT) linear_kernel(const __grid_constant__ LinearPlan p) {
  __shared__ float sums[WARPS][16 * TILES][8 * COLUMNS + 1];
  constexpr int kScaleWords = 8 * Unit<GROUP>::kWords;  // of a unit's tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int chunks = static_cast<int>(chunks_of(p.w.inputs)), units = (chunks + 1) / 2;
  const int all = p.rows / p.parts, first = static_cast<int>(blockIdx.y) * p.per, mine = min(p.per, all - first);
  const long long tile = static_cast<long long>(blockIdx.x) * TILES, last = tiles_of(p.w.outputs) - 1;
  pdl_launch_dependents();
  if (mine <= 0) return;

  // column j of the block's: part j / mine of row first + j % mine
  const uint16_t* x[COLUMNS];
#pragma unroll
  for (int t = 0; t < COLUMNS; ++t) {
    const int j = t * 8 + g, row = j < mine * p.parts ? j / mine * all + first + j % mine : first;
    x[t] = static_cast<const uint16_t*>(p.x) + static_cast<long long>(row) * p.ld + c * 8;
  }
  const uint4* codes[TILES];
  const uint32_t* scales[TILES];
#pragma unroll
  for (int n = 0; n < TILES; ++n) {
    const long long at = min(tile + n, last);  // (one that is not there is computed like the last and not stored)
    codes[n] = static_cast<const uint4*>(p.w.codes) + at * chunks * 32 + lane;
    scales[n] = static_cast<const uint32_t*>(p.w.scales) + at * tile_scales(p.w.inputs, GROUP) / 2 +
                g * (GROUP == 32 ? 2 : 1);
  }
  float total[TILES][COLUMNS][4];
#pragma unroll
  for (int n = 0; n < TILES; ++n)
#pragma unroll
    for (int t = 0; t < COLUMNS; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[n][t][i] = 0.0f;
  pdl_wait();
  const int whole = static_cast<int>(p.w.inputs / 128);  // units that are
  Unit<GROUP> ring[2][TILES];
  auto load = [&](Unit<GROUP>* u, int unit) {
    if (unit < whole) {
#pragma unroll
      for (int n = 0; n < TILES; ++n)
        load_unit<GROUP, true>(u[n], codes[n] + static_cast<long long>(unit) * 64,
                               scales[n] + static_cast<long long>(unit) * kScaleWords);
    }
  };
  load(ring[0], warp);
  int unit = warp;
  for (; unit < whole; unit += 2 * WARPS) {
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
      const int now = unit + slot * WARPS;
      if (now >= whole) break;
      load(ring[slot ^ 1], now + WARPS);
      multiply_units<HALF, GROUP, COLUMNS, TILES, true>(ring[slot], x, now * 128LL, 0, p.w.scale_dtype, total);
    }
  }
  if (whole < units && whole % WARPS == warp) {  // less than a unit is left
    const long long k = whole * 128LL;
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      const uint4* from = codes[n] + static_cast<long long>(whole) * 64;
      const uint32_t* by = scales[n] + static_cast<long long>(whole) * kScaleWords;
      if (2 * whole + 1 < chunks) load_unit<GROUP, true>(ring[0][n], from, by);
      else load_unit<GROUP, false>(ring[0][n], from, by);
    }
    multiply_units<HALF, GROUP, COLUMNS, TILES, false>(ring[0], x, k, p.w.inputs - k - c * 8, p.w.scale_dtype, total);
  }
#pragma unroll
  for (int n = 0; n < TILES; ++n)
#pragma unroll
    for (int t = 0; t < COLUMNS; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[warp][n * 16 + g + i / 2 * 8][t * 8 + 2 * c + i % 2] = total[n][t][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * TILES * mine; i += 32 * WARPS) {
    const int n = i % (16 * TILES), r = i / (16 * TILES);
    float y = 0.0f;
    for (int part = 0; part < p.parts; ++part)
#pragma unroll
      for (int v = 0; v < WARPS; ++v) y += sums[v][n][part * mine + r];
    if (tile * 16 + n < p.w.outputs) store_from_f32(p.out, (first + r) * p.out_ld + tile * 16 + n, p.out_dtype, y);
  }
}

// x in a form that the products can read: float32 as three bfloat16 parts, 16-bit
// rows that do not lie on 16 bytes as they are, in rows of ld elements.
__global__ void __launch_bounds__(256) arrange_kernel(const void* x, int dtype, long long ld, long long rows,
                                                      long long inputs, uint16_t* to, long long to_ld) {
  pdl_launch_dependents();
  pdl_wait();
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= rows * inputs) return;
  const long long r = at / inputs, k = at % inputs;
  if (dtype == CB_F32) {
    float v = static_cast<const float*>(x)[r * ld + k];
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      const __nv_bfloat16 h = __float2bfloat16_rz(v);  // (towards zero: 8 bits each, and nothing becomes infinite)
      to[(part * rows + r) * to_ld + k] = __bfloat16_as_ushort(h);
      v -= __bfloat162float(h);
      if (!isfinite(__bfloat162float(h))) v = 0.0f;  // an infinity or NaN is in the first part alone
    }
  } else {
    to[r * to_ld + k] = static_cast<const uint16_t*>(x)[r * ld + k];
  }
}

// ---- making and unmaking weights -----------------------------------------------

// One word of a lane for each thread; outputs and inputs beyond the last have code 8, zero.
__global__ void __launch_bounds__(256) pack_kernel(const uint8_t* codes, const uint16_t* scales, const cb_weights4 w) {
  const long long chunks = chunks_of(w.inputs), words = tiles_of(w.outputs) * chunks * 128;
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (at < words) {
    const int s = at % 4, lane = at / 4 % 32;
    const long long tile = at / 128 / chunks, chunk = at / 128 % chunks;
    const long long k = chunk * 64 + s / 2 * 32 + lane % 4 * 8 + s % 2 * 4;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long n = tile * 16 + lane / 4 + i % 2 * 8, from = k + i / 2 * 2;
      const uint32_t byte = n < w.outputs && from < w.inputs ? codes[n * (w.inputs / 2) + from / 2] : 0x88u;
      word |= (byte & 15u) << 4 * i | byte >> 4 << (16 + 4 * i);
    }
    const_cast<uint32_t*>(static_cast<const uint32_t*>(w.codes))[at] = word;
  }
  // scales of outputs and groups that do not exist are zero
  const long long per = tile_scales(w.inputs, w.group), all = tiles_of(w.outputs) * per;
  const long long groups = w.inputs / w.group;
  for (long long i = at; i < all; i += static_cast<long long>(gridDim.x) * 256) {
    const long long tile = i / per, in = i % per;
    const long long row = w.group == 32 ? in % 32 / 4 + in % 2 * 8 : in % 16 / 2 + in % 2 * 8;
    const long long group = w.group == 32 ? in / 32 * 2 + in % 4 / 2 : in / 16, n = tile * 16 + row;
    const_cast<uint16_t*>(static_cast<const uint16_t*>(w.scales))[i] =
        n < w.outputs && group < groups ? scales[n * groups + group] : 0;
  }
}

// A warp to 16 outputs x 64 inputs.  Bound by its instructions before its stores: the
// codes come out of a word as bytes, by whose place a float's bits are made (2^23 + code),
// and the group and the strides are known when it is compiled or computed once (4096 x
// 14336 to bfloat16: 24.9 us, 5.9 TB/s; with divisions and a conversion each, 41).
template <int GROUP, int ITEM>
__global__ void __launch_bounds__(256) dequantise_kernel(const cb_weights4 w, void* out, int dtype, long long ld,
                                                         int wide) {
  const int chunks = static_cast<int>(chunks_of(w.inputs));
  const long long block = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (block >= tiles_of(w.outputs) * chunks) return;
  const int lane = threadIdx.x & 31, g = lane / 4, c = lane % 4;
  const int tile = static_cast<int>(static_cast<unsigned>(block) / static_cast<unsigned>(chunks));
  const int chunk = static_cast<int>(block) - tile * chunks;
  const uint4 w4 = __ldcs(static_cast<const uint4*>(w.codes) + block * 32 + lane);
  const uint32_t words[4] = {w4.x, w4.y, w4.z, w4.w};
  const uint32_t* from = static_cast<const uint32_t*>(w.scales) + tile * tile_scales(w.inputs, GROUP) / 2;
  uint32_t both[2];
  if (GROUP == 32) {
    const uint2 two = __ldg(reinterpret_cast<const uint2*>(from) + chunk * 8LL + g);
    both[0] = two.x;
    both[1] = two.y;
  } else {
    both[0] = both[1] = __ldg(from + (GROUP == 128 ? chunk / 2 : chunk) * 8LL + g);
  }
  const long long k = chunk * 64LL + c * 8, n = tile * 16LL + g;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (k + half * 32 >= w.inputs) break;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (n + which * 8 >= w.outputs) continue;
      const float s = scale_of(both[half] >> (16 * which) & 0xffffu, w.scale_dtype);
      // pairs `which` and `which` + 2 of both words: even elements in the low halves
      float v[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t word = words[2 * half + i] >> (4 * which);
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          const uint32_t two = word >> (8 * pair) & 0x000f000fu;
          v[4 * i + 2 * pair] = (__uint_as_float((two & 0xffffu) | 0x4b000000u) - 8388616.0f) * s;
          v[4 * i + 2 * pair + 1] = (__uint_as_float(two >> 16 | 0x4b000000u) - 8388616.0f) * s;
        }
      }
      const long long at = (n + which * 8) * ld + k + half * 32;
      if (!wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) store_from_f32(out, at + i, dtype, v[i]);
      } else if (ITEM == 4) {
        float* to = static_cast<float*>(out) + at;
        __stcs(reinterpret_cast<float4*>(to), make_float4(v[0], v[1], v[2], v[3]));
        __stcs(reinterpret_cast<float4*>(to) + 1, make_float4(v[4], v[5], v[6], v[7]));
      } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (dtype == CB_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            h[i] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            h[i] = *reinterpret_cast<const uint32_t*>(&b);
          }
        }
        __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at), make_uint4(h[0], h[1], h[2], h[3]));
      }
    }
  }
}

// A warp to a group: s = rn(max |w| / 7), q = rne(w / s) within [-8, 7].
__global__ void __launch_bounds__(256) quantise_kernel(const void* weight, int dtype, long long ld, const cb_weights4 w,
                                                       uint8_t* codes, uint16_t* scales) {
  const long long groups = w.inputs / w.group;
  const long long at = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (at >= w.outputs * groups) return;
  const int lane = threadIdx.x & 31;
  const long long n = at / groups, k = at % groups * w.group;
  float largest = 0.0f;
  bool fine = true;
  for (int i = lane; i < w.group; i += 32) {
    const float v = load_as_f32(weight, n * ld + k + i, dtype);
    fine = fine && isfinite(v);
    largest = fmaxf(largest, fabsf(v));
  }
  largest = warp_max(largest);
  fine = __all_sync(0xffffffffu, fine);
  // (a group with an infinity or a NaN has a NaN scale: its products are NaN, not wrong)
  const float s = round_to(fine ? largest / 7.0f : NAN, w.scale_dtype);
  if (lane == 0)
    scales[at] = w.scale_dtype == CB_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(s))
                                          : __half_as_ushort(__float2half_rn(s));
  for (int i = 2 * lane; i < w.group; i += 64) {
    uint32_t byte = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = load_as_f32(weight, n * ld + k + i + j, dtype);
      const float q = s > 0.0f && fine ? fminf(fmaxf(rintf(v / s), -8.0f), 7.0f) : 0.0f;
      byte |= static_cast<uint32_t>(static_cast<int>(q) + 8) << 4 * j;
    }
    codes[n * (w.inputs / 2) + (k + i) / 2] = static_cast<uint8_t>(byte);
  }
}

int weights_check(const cb_weights4& w, const char* who) {
  CB_REQUIRE(w.group == 32 || w.group == 64 || w.group == 128, "%s: groups of 32, 64 or 128 (got %d)", who, w.group);
  CB_REQUIRE(w.scale_dtype == CB_BF16 || w.scale_dtype == CB_F16, "%s: scales must be bfloat16 or float16", who);
  CB_REQUIRE(w.outputs >= 1 && w.inputs >= w.group && w.inputs % w.group == 0 && w.outputs < (1LL << 31) &&
                 w.inputs < (1LL << 31) && tiles_of(w.outputs) * chunks_of(w.inputs) < (1LL << 31),
             "%s: %lld outputs of %lld inputs in groups of %d", who, w.outputs, w.inputs, w.group);
  return CB_OK;
}

int weights_and_pools_check(const cb_weights4& w, const char* who) {
  const int status = weights_check(w, who);
  if (status != CB_OK) return status;
  CB_REQUIRE(w.codes != nullptr && w.scales != nullptr && reinterpret_cast<uintptr_t>(w.codes) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(w.scales) % 16 == 0,
             "%s: codes and scales must be given, aligned to 16 bytes", who);
  return CB_OK;
}

bool on_its_type(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == CB_F32 ? 4 : 2) == 0; }

bool needs_arranging(const cb_linear4_args& a) {
  return a.dtype == CB_F32 || reinterpret_cast<uintptr_t>(a.x) % 16 != 0 || (a.rows > 1 && a.ld % 8 != 0);
}

template <int N>
using is = std::integral_constant<int, N>;

template <typename F>
int with_columns(int columns, F f) {
  if (columns <= 1) return f(is<1>{});
  if (columns == 2) return f(is<2>{});
  if (columns == 3) return f(is<3>{});
  return f(is<4>{});
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

long long cb_weights4_code_bytes(const cb_weights4* weights) {
  if (weights == nullptr || weights_check(*weights, "cb_weights4_code_bytes") != CB_OK) return 0;
  return tiles_of(weights->outputs) * chunks_of(weights->inputs) * kBlockBytes;
}

long long cb_weights4_scale_bytes(const cb_weights4* weights) {
  if (weights == nullptr || weights_check(*weights, "cb_weights4_scale_bytes") != CB_OK) return 0;
  return tiles_of(weights->outputs) * tile_scales(weights->inputs, weights->group) * 2;
}

int cb_weights4_quantise(const cb_weights4* weights, const void* weight, int dtype, long long ld, void* codes,
                         void* scales, cb_stream_t stream) {
  CB_REQUIRE(weights != nullptr, "cb_weights4_quantise: null arguments");
  const cb_weights4& w = *weights;
  const int status = weights_check(w, "cb_weights4_quantise");
  if (status != CB_OK) return status;
  CB_REQUIRE(dtype == CB_F32 || dtype == CB_BF16 || dtype == CB_F16,
             "cb_weights4_quantise: weights must be float32, bfloat16 or float16");
  CB_REQUIRE(weight != nullptr && codes != nullptr && scales != nullptr, "cb_weights4_quantise: a null pointer");
  CB_REQUIRE(on_its_type(weight, dtype) && on_its_type(scales, w.scale_dtype),
             "cb_weights4_quantise: weight and scales must be aligned to their types");
  const long long blocks = (w.outputs * (w.inputs / w.group) + 7) / 8;
  CB_REQUIRE(blocks < (1LL << 31), "cb_weights4_quantise: %lld outputs of %lld inputs", w.outputs, w.inputs);
  quantise_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      weight, dtype, ld, w, static_cast<uint8_t*>(codes), static_cast<uint16_t*>(scales));
  return check_launch("cb_weights4_quantise");
}

int cb_weights4_pack(const cb_weights4* weights, const void* codes, const void* scales, cb_stream_t stream) {
  CB_REQUIRE(weights != nullptr, "cb_weights4_pack: null arguments");
  const cb_weights4& w = *weights;
  const int status = weights_and_pools_check(w, "cb_weights4_pack");
  if (status != CB_OK) return status;
  CB_REQUIRE(codes != nullptr && scales != nullptr, "cb_weights4_pack: a null pointer");
  CB_REQUIRE(on_its_type(scales, w.scale_dtype), "cb_weights4_pack: scales must be aligned to their type");
  const long long blocks = (tiles_of(w.outputs) * chunks_of(w.inputs) * 128 + 255) / 256;
  CB_REQUIRE(blocks < (1LL << 31), "cb_weights4_pack: %lld outputs of %lld inputs", w.outputs, w.inputs);
  pack_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(codes), static_cast<const uint16_t*>(scales), w);
  return check_launch("cb_weights4_pack");
}

int cb_weights4_dequantise(const cb_weights4* weights, void* out, int dtype, long long ld, cb_stream_t stream) {
  CB_REQUIRE(weights != nullptr, "cb_weights4_dequantise: null arguments");
  const cb_weights4& w = *weights;
  const int status = weights_and_pools_check(w, "cb_weights4_dequantise");
  if (status != CB_OK) return status;
  CB_REQUIRE(dtype == CB_F32 || dtype == CB_BF16 || dtype == CB_F16,
             "cb_weights4_dequantise: out must be float32, bfloat16 or float16");
  CB_REQUIRE(out != nullptr && ld >= w.inputs, "cb_weights4_dequantise: rows of %lld elements", ld);
  CB_REQUIRE(on_its_type(out, dtype), "cb_weights4_dequantise: out must be aligned to its type");
  const int item = dtype == CB_F32 ? 4 : 2;
  const int wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld * item % 16 == 0;
  const unsigned blocks = static_cast<unsigned>((tiles_of(w.outputs) * chunks_of(w.inputs) + 7) / 8);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto group) {
    if (item == 4) dequantise_kernel<group.value, 4><<<blocks, 256, 0, s>>>(w, out, dtype, ld, wide);
    else dequantise_kernel<group.value, 2><<<blocks, 256, 0, s>>>(w, out, dtype, ld, wide);
  };
  if (w.group == 32) go(std::integral_constant<int, 32>{});
  else if (w.group == 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
  return check_launch("cb_weights4_dequantise");
}

long long cb_linear4_scratch(const cb_linear4_args* args) {
  if (args == nullptr || args->rows <= 0 || !needs_arranging(*args)) return 0;
  return args->rows * (args->dtype == CB_F32 ? 3 : 1) * args->weights.inputs * 2;
}

int cb_linear4(const cb_linear4_args* args, void* scratch, cb_stream_t stream) {
  CB_REQUIRE(args != nullptr, "cb_linear4: null arguments");
  const cb_linear4_args& a = *args;
  const int status = weights_and_pools_check(a.weights, "cb_linear4");
  if (status != CB_OK) return status;
  CB_REQUIRE(a.dtype == CB_F32 || a.dtype == CB_BF16 || a.dtype == CB_F16,
             "cb_linear4: x must be float32, bfloat16 or float16");
  const int parts = a.dtype == CB_F32 ? 3 : 1, most = kColumnTiles * 8 / parts;  // rows that a block can take
  CB_REQUIRE(a.rows >= 0 && a.rows <= 65535LL * most, "cb_linear4: %lld rows, at most %lld are taken", a.rows,
             65535LL * most);
  if (a.rows == 0) return CB_OK;
  CB_REQUIRE(a.x != nullptr && a.out != nullptr, "cb_linear4: a null pointer");
  CB_REQUIRE(on_its_type(a.x, a.dtype) && on_its_type(a.out, a.dtype),
             "cb_linear4: x and out must be aligned to their type");
  CB_REQUIRE(a.rows == 1 || a.out_ld >= a.weights.outputs || -a.out_ld >= a.weights.outputs,
             "cb_linear4: rows of %lld outputs, %lld apart, share memory", a.weights.outputs, a.out_ld);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  LinearPlan p = {};
  p.w = a.weights;
  p.x = a.x;
  p.ld = a.ld;
  p.parts = parts;
  p.rows = static_cast<int>(a.rows * p.parts);
  p.out = a.out;
  p.out_dtype = a.dtype;
  p.out_ld = a.out_ld;
  if (needs_arranging(a)) {
    CB_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0,
               "cb_linear4: %lld bytes of scratch are needed, aligned to 16", cb_linear4_scratch(args));
    const long long blocks = (a.rows * a.weights.inputs + 255) / 256;
    CB_REQUIRE(blocks < (1LL << 31), "cb_linear4: %lld rows of %lld", a.rows, a.weights.inputs);
    launch(arrange_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, true, a.x, a.dtype, a.ld, a.rows,
           a.weights.inputs, static_cast<uint16_t*>(scratch), a.weights.inputs);
    const int arranged = check_launch("cb_linear4");
    if (arranged != CB_OK) return arranged;
    p.x = scratch;
    p.ld = a.weights.inputs;
  }
  const int launches = static_cast<int>((a.rows + most - 1) / most);
  p.per = static_cast<int>((a.rows + launches - 1) / launches);
  return with_columns((p.per * p.parts + 7) / 8, [&](auto columns) {
    constexpr int C = columns.value;
    const long long tiles = tiles_of(a.weights.outputs);
    // The form of a block: its tiles, its warps, and how many are on an SM.  Few tiles
    // have many warps each, so that each chain of loads and products is short (tiles of
    // 5632 inputs on 128 SMs, 15 columns: 16 warps 7.0 us, 8 warps 9.7; 256 tiles of 14336
    // inputs, one column: 8.9 and 11.4); many have few, which wait for few others (896
    // tiles of 4096 inputs, one column: 4 warps, 7 blocks an SM 8.9, 8 warps, 4 blocks 9.9),
    // and from there on two tiles share the rows of x as long as their sums fit the
    // registers (8016 tiles: one column 55 us and 60 with 8 warps, 16 columns 77 and 91;
    // one tile to a block 56 and 99).
    auto go = [&](auto group, auto count, auto warps, auto resident) {
      constexpr int T = count.value, WARPS = warps.value, RESIDENT = resident.value;
      const dim3 grid(static_cast<unsigned>((tiles + T - 1) / T), static_cast<unsigned>(launches));
      if (a.dtype == CB_F16)
        launch(linear_kernel<true, group.value, C, T, WARPS, RESIDENT>, grid, dim3(32 * WARPS), 0, s, true, p);
      else
        launch(linear_kernel<false, group.value, C, T, WARPS, RESIDENT>, grid, dim3(32 * WARPS), 0, s, true, p);
      return check_launch("cb_linear4");
    };
    auto by_tiles = [&](auto group) {
      const long long all = tiles * launches, sms = sm_count();
      if (all <= sms) return go(group, is<1>{}, is<16>{}, is<1>{});
      if constexpr (C > 2) {  // (32 rows: 896 tiles 26 us, with 8 warps 30; 256 tiles are not a wave of these)
        if (all <= 2 * sms) return go(group, is<1>{}, is<8>{}, is<2>{});
        return go(group, is<1>{}, is<4>{}, is<4>{});
      } else {
        if (all <= 2 * sms) return go(group, is<1>{}, is<16>{}, is<2>{});
        if (all <= 3 * sms) return go(group, is<1>{}, is<8>{}, is<3>{});
        if constexpr (C == 2) {  // (563 tiles: one to a block 10.0 us, two 12.7; 896 tiles: 18.3 and 13.1)
          if (all <= 5 * sms) return go(group, is<1>{}, is<4>{}, is<5>{});
          return go(group, is<2>{}, is<4>{}, is<4>{});
        } else {
          if (all <= 4 * sms) return go(group, is<1>{}, is<8>{}, is<4>{});
          if (all >= 16 * sms) return go(group, is<2>{}, is<4>{}, is<6>{});
          // seven blocks an SM have more registers, eight may save a wave (1184 tiles of 3584 inputs: 12.1 and
          // 9.1 us; 896 of 4096: 8.9 and 10.0)
          const bool saves = (all + 7 * sms - 1) / (7 * sms) > (all + 8 * sms - 1) / (8 * sms);
          return saves ? go(group, is<1>{}, is<4>{}, is<8>{}) : go(group, is<1>{}, is<4>{}, is<7>{});
        }
      }
    };
    if (a.weights.group == 32) return by_tiles(is<32>{});
    if (a.weights.group == 64) return by_tiles(is<64>{});
    return by_tiles(is<128>{});
  });
}

}  // extern "C"
