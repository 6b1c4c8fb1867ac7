// A projection in 8-bit integers, a scale for each token and each output
// channel, for gfx950:
//   s_m = max_k |x_mk| / 127,  q_mk = rint(127 x_mk / max_k |x_mk|),
//   y_mn = (sum_k q_mk w_nk) s_m t_n,
// the sum a whole number in 32 bits (K is at most 131,072).
//
// Layout.  Weights and codes lie in tiles of 16 rows by 64 inputs, 1 KiB in
// the order in which the matrix instruction takes them: the 16 bytes at 16 l
// are row l % 16, inputs 16 (l / 16) ... + 15.  A wave's load of a tile is one
// run of 1 KiB, a copy of it to LDS needs no rearranging, and a read from LDS
// meets no bank twice.  Inputs are filled up to a multiple of 128 by zeros.
#include "m2r_device.h"
#include "m2r_abi_util.h"

#include <initializer_list>

namespace m2r {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kTile = 1024;
static int64_t padded_inputs(int64_t K) { return (K + 127) / 128 * 128; }
static int64_t row_tiles(int64_t rows) { return (rows + 15) / 16; }

// ---------------------------------------------------------------- codes of rows
// The code of x is rint(127 x / top), ties to even, as in exact arithmetic.
// With 11 significant bits in x and top (8 in bfloat16), 127 x / top is either
// half of an odd number up to 253 or at least 2^-19 of its value away from any
// such number: |254 x - (2 k + 1) top| is 0 or a unit of a number below 2^19
// units.  x / top in two roundings is within 2^-23 of its value; rounded to 21
// bits it is the tie where there is one, and on the right side of it otherwise.
struct RowArgs {
  const uint16_t* x;
  int64_t stride, rows, K, Kp;
  uint8_t* tiles;
  float* scale;
};

template <bool BF16>
__device__ __forceinline__ float half_value(uint32_t bits) {
  return BF16 ? __builtin_bit_cast(float, bits << 16) : h2f((uint16_t)bits);
}

template <bool BF16>
__device__ __forceinline__ uint32_t code_of(uint32_t bits, float factor, int shift) {
  float v = half_value<BF16>(bits);
  if (BF16) v = __builtin_ldexpf(v, shift);     // binary32's range is bfloat16's: relative to top
  const float q = v * factor;
  const float snapped = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, q) + 4u) & ~7u);
  return __builtin_bit_cast(uint32_t, snapped + 0x1.8p23f);   // the low byte
}

// A wave a row; 16 inputs of a lane are 16 bytes of a tile.
template <bool BF16>
__global__ __launch_bounds__(256) void k_int8_rows(RowArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const uint16_t* x = a.x + row * a.stride;
  uint32_t top = 0;
  for (int64_t k = lane; k < a.K; k += 64) {
    const uint32_t v = x[k] & 0x7fffu;
    top = top > v ? top : v;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t v = (uint32_t)__shfl_xor((int)top, d);
    top = top > v ? top : v;
  }
  const bool finite = top < (BF16 ? 0x7f80u : 0x7c00u);
  const float largest = half_value<BF16>(top);
  int shift = 0;
  if (BF16 && finite && top) shift = -__builtin_amdgcn_frexp_expf(largest);
  const float factor = finite && top ? 127.f / (BF16 ? __builtin_ldexpf(largest, shift) : largest) : 0.f;
  if (lane == 0) a.scale[row] = finite ? largest / 127.f : __builtin_nanf("");
  uint8_t* out = a.tiles + (row >> 4) * 16 * a.Kp + (row & 15) * 16;
  for (int64_t k0 = lane * 16; k0 < a.Kp; k0 += 1024) {
    uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t bits = finite && k0 + j < a.K ? x[k0 + j] : 0u;
      word[j >> 2] |= (code_of<BF16>(bits, factor, shift) & 0xffu) << (8 * (j & 3));
    }
    *(u32x4*)(out + (k0 >> 6) * kTile + (k0 >> 4 & 3) * 256) = u32x4{word[0], word[1], word[2], word[3]};
  }
}

// ---------------------------------------------------------------- the product
struct ProductArgs {
  const uint8_t *x, *w;          // tiles
  const float *xs, *ws;          // scales of rows and channels
  void* y;
  int64_t ys, M, N, Kp;
  int64_t channel_groups;
};

// sum * token * channel in binary32: the smaller scale first, so that no
// product on the way leaves binary32's range unless the value does (an integer
// times a subnormal scale is exact).  A NaN scale gives NaN.
__device__ __forceinline__ float scaled(int sum, float token, float channel) {
  const bool less = token < channel;
  return (float)sum * (less ? token : channel) * (less ? channel : token);
}

template <int DTYPE>
__device__ __forceinline__ void store_value(void* y, int64_t at, float v) {
  if constexpr (DTYPE == 0) ((uint16_t*)y)[at] = f2h(v);
  else if constexpr (DTYPE == 1) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    ((uint16_t*)y)[at] = v != v ? (uint16_t)(u >> 16 | 0x40) : (uint16_t)((u + 0x7fffu + (u >> 16 & 1)) >> 16);
  } else ((float*)y)[at] = v;
}

// A wave takes 16 rows by 16 channels.
template <int DTYPE>
__global__ __launch_bounds__(256) void k_int8_product(ProductArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t nt = (blockIdx.x % a.channel_groups) * 4 + wave, mt = blockIdx.x / a.channel_groups;
  if (nt * 16 >= a.N) return;
  const uint8_t* w = a.w + nt * 16 * a.Kp + lane * 16;
  const uint8_t* x = a.x + mt * 16 * a.Kp + lane * 16;
  i32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int64_t k = 0; k < a.Kp / 64; ++k)
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(w + k * kTile), *(const i32x4*)(x + k * kTile), acc, 0, 0,
                                                0);
  const int64_t m = mt * 16 + (lane & 15), n = nt * 16 + 4 * (lane >> 4);
  if (m >= a.M) return;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.N) store_value<DTYPE>(a.y, m * a.ys + n + r, scaled(acc[r], a.xs[m], a.ws[n + r]));
}

}  // namespace m2r

using namespace m2r;

static int int8_rows(const void* x, int dtype, int64_t stride, int64_t rows, int64_t K, uint8_t* tiles, float* scale,
                     hipStream_t stream) {
  const RowArgs a{(const uint16_t*)x, stride, rows, K, padded_inputs(K), tiles, scale};
  const dim3 grid((unsigned)((rows + 3) / 4)), block(256);
  if (dtype == 0) hipLaunchKernelGGL((k_int8_rows<false>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((k_int8_rows<true>), grid, block, 0, stream, a);
  return m2r_check(hipGetLastError(), "int8 rows launch");
}

static int int8_limits(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0) return m2r_fail("int8: non-positive shape");
  if (rows > (int64_t)1 << 24 || K > 131072) return m2r_fail("int8: size limits");
  return 0;
}

extern "C" int64_t m2r_int8_tiles_bytes(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0) return 0;
  return row_tiles(rows) * 16 * padded_inputs(K);
}

extern "C" int m2r_int8_quantize(const void* x, int dtype, int64_t x_stride, void* tiles, float* scale, int64_t rows,
                                 int64_t K, hipStream_t stream) {
  if (int rc = int8_limits(rows, K)) return rc;
  if (dtype < 0 || dtype > 1) return m2r_fail("int8: x must be binary16 or bfloat16");
  if (!x || !tiles || !scale) return m2r_fail("int8: null pointer");
  if (x_stride < 0) return m2r_fail("int8: negative stride");
  if ((uintptr_t)tiles & 15) return m2r_fail("int8: tiles must be 16-byte aligned");
  return int8_rows(x, dtype, x_stride, rows, K, (uint8_t*)tiles, scale, stream);
}

extern "C" int64_t m2r_int8_linear_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return m2r_int8_tiles_bytes(M, K) + 4 * M;
}

extern "C" int m2r_int8_linear(const void* x, int x_dtype, int64_t x_stride, const void* w_tiles, const float* w_scale,
                               void* y, int y_dtype, int64_t y_stride, int64_t M, int64_t N, int64_t K, void* workspace,
                               int64_t workspace_bytes, hipStream_t stream) {
  if (N <= 0) return m2r_fail("int8: non-positive shape");
  if (int rc = int8_limits(M, K)) return rc;
  if (N > (int64_t)1 << 24) return m2r_fail("int8: size limits");
  if (x_dtype < 0 || x_dtype > 1) return m2r_fail("int8: x must be binary16 or bfloat16");
  if (y_dtype < 0 || y_dtype > 2) return m2r_fail("int8: y must be binary16, bfloat16 or binary32");
  for (const void* p : {x, w_tiles, (const void*)w_scale, (const void*)y, (const void*)workspace})
    if (!p) return m2r_fail("int8: null pointer");
  if (x_stride < 0) return m2r_fail("int8: negative stride");
  if (y_stride < N) return m2r_fail("int8: rows overlap");
  if ((uintptr_t)w_tiles & 15) return m2r_fail("int8: tiles must be 16-byte aligned");
  if ((uintptr_t)workspace & 15 || workspace_bytes < m2r_int8_linear_workspace(M, N, K))
    return m2r_fail("int8: workspace too small or not 16-byte aligned");
  uint8_t* codes = (uint8_t*)workspace;
  float* scale = (float*)(codes + m2r_int8_tiles_bytes(M, K));
  if (int rc = int8_rows(x, x_dtype, x_stride, M, K, codes, scale, stream)) return rc;
  const int64_t groups = (N + 63) / 64;
  if (groups * row_tiles(M) > 0x7fffffff) return m2r_fail("int8: grid limits exceeded");
  const ProductArgs a{codes, (const uint8_t*)w_tiles, scale, w_scale, y, y_stride, M, N, padded_inputs(K), groups};
  const dim3 grid((unsigned)(groups * row_tiles(M))), block(256);
  if (y_dtype == 0) hipLaunchKernelGGL((k_int8_product<0>), grid, block, 0, stream, a);
  else if (y_dtype == 1) hipLaunchKernelGGL((k_int8_product<1>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((k_int8_product<2>), grid, block, 0, stream, a);
  return m2r_check(hipGetLastError(), "int8 product launch");
}
