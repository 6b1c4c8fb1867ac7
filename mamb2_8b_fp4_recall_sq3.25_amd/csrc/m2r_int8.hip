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
// Of 32 channels the two tiles of weights take four each in turn, so that the
// lane that holds rows 4 g ... + 3 of both products holds channels 8 g ... + 7.
//
// One launch forms the rows' codes, one multiplies; up to four rows have both in
// one.  Times in a graph of calls (us; reads alone reach 7.0 TB/s, a large copy
// 5.0, a library product of 8,192 cubed in these types 2.2 POP/s):
//   1 row, 4,096 -> 18,560      18   4.3 TB/s: memory, a launch's start and end (15 where the
//                                    weights are in the last-level cache)
//   64 rows, 8,192 -> 4,096     20   1.8 TB/s: two launches, operands' way from L2 (15 likewise)
//   24 rows, 4,096 -> 256,000  200   5.4 TB/s: memory
//   901 rows, 8,192 -> 4,096    43   1.4 POP/s: a block of 128 x 128 a CU, whose
//                                    operands come from L2 at half of what a CU can take
//   2,048 rows, 4,096 -> 18,560 146  2.1 POP/s: see tile_block
#include "m2r_device.h"
#include "m2r_abi_util.h"
#include "m2r_tile.h"

#include <initializer_list>

namespace m2r {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 1024;
static int64_t padded_inputs(int64_t K) { return (K + 127) / 128 * 128; }
static int64_t row_tiles(int64_t rows) { return (rows + 15) / 16; }
static int64_t channel_tiles(int64_t channels) { return (channels + 31) / 32 * 2; }

// ---------------------------------------------------------------- codes of rows
// The code of x is rint(127 x / top), ties to even, as in exact arithmetic.
// With 11 significant bits in x and top (8 in bfloat16), 127 x / top is either
// half of an odd number up to 253 or at least 2^-19 of its value away from any
// such number: |254 x - (2 k + 1) top| is 0 or a unit of a number below 2^19
// units.  x (127 / top) in two roundings is within 2^-23 of its value; rounded
// to 21 bits it is the tie where there is one, and on the right side of it
// otherwise.
struct RowArgs {
  const uint16_t* x;
  int64_t stride, rows, K, Kp;
  uint8_t* tiles;
  float* scale;
  uint32_t* clear;       // words to set to 0 for the product that follows
  int64_t clears;
  int channels;          // 1: rows are output channels of weights
  int whole;             // 1: rows of whole sixteens at 16-byte boundaries
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

struct Chunk { u16x8 h[2]; };   // 16 inputs of a row

// Inputs 16 c ... + 15 of a row, zeros from K on.  WHOLE: rows of whole sixteens
// at 16-byte boundaries, read without a branch.
template <bool WHOLE>
__device__ __forceinline__ Chunk load_chunk(const RowArgs& a, const uint16_t* x, int c) {
  Chunk v;
  const int last = (int)(a.K >> 4);
  if constexpr (WHOLE) {
    const auto row = __builtin_amdgcn_make_buffer_rsrc((void*)x, 0, (int)(2 * a.K), 0x00027000);   // zeros past its end
    v.h[0] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(row, 32 * c, 0, 0));
    v.h[1] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(row, 32 * c + 16, 0, 0));
  } else if (c < last) {
    __builtin_memcpy(&v, x + 16 * (int64_t)c, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v.h[j >> 3][j & 7] = 16 * (int64_t)c + j < a.K ? x[16 * (int64_t)c + j] : (uint16_t)0;
  }
  return v;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 largest_of(const Chunk& v, u16x2 top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const u16x2 pair = {(uint16_t)(v.h[j >> 2][2 * (j & 3)] & 0x7fff), (uint16_t)(v.h[j >> 2][2 * (j & 3) + 1] & 0x7fff)};
    top = __builtin_elementwise_max(top, pair);
  }
  return top;
}
__device__ __forceinline__ uint32_t wave_largest(u16x2 pair) {
  uint32_t top = pair[0] > pair[1] ? pair[0] : pair[1];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t v = (uint32_t)__shfl_xor((int)top, d);
    top = top > v ? top : v;
  }
  return top;
}
struct RowScale {
  float factor, scale;   // a row that is not finite has the scale NaN, and codes that do not matter
  int shift;
};
template <bool BF16>
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  RowScale s{};
  const bool finite = top < (BF16 ? 0x7f80u : 0x7c00u);
  const float largest = half_value<BF16>(top);
  if (BF16 && finite && top) s.shift = -__builtin_amdgcn_frexp_expf(largest);
  s.factor = finite && top ? 127.f / (BF16 ? __builtin_ldexpf(largest, s.shift) : largest) : 0.f;
  s.scale = finite ? largest / 127.f : __builtin_nanf("");
  return s;
}
template <bool BF16>
__device__ __forceinline__ u32x4 codes_of(const Chunk& v, const RowScale& s) {
  u32x4 word;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = code_of<BF16>(v.h[q >> 1][4 * (q & 1) + j], s.factor, s.shift);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    word[q] = lo | hi;
  }
  return word;
}

// A workgroup a row, 16 inputs a thread at a time; the first kHeld of a thread
// stay in registers between the two passes over the row.  The 16 rows of a tile
// are workgroups of one XCD, whose L2 puts their pieces of a line together.
// (A wave a row, eight rows a workgroup, which fills whole lines by itself, takes
// longer: 64 rows of 8,192 inputs 9 us against 4, a row's arithmetic in one wave.)
constexpr int kHeld = 4;
constexpr int kFusedInputs = 8192;   // of a row whose codes k_int8_few forms itself
template <bool BF16, bool WHOLE>
__global__ __launch_bounds__(256) void k_int8_rows(RowArgs a) {
  __shared__ uint32_t tops[4];
  const int tid = threadIdx.x;
  for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < a.clears; i += (int64_t)gridDim.x * 256) a.clear[i] = 0;
  const uint32_t turn = blockIdx.x >> 3;
  const int64_t row = ((int64_t)(turn >> 4) * 8 + (blockIdx.x & 7)) * 16 + (turn & 15);
  if (row >= a.rows) return;
  const uint16_t* x = a.x + row * a.stride;
  const int chunks = (int)(a.Kp / 16);
  Chunk held[kHeld] = {};
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (256 * i < chunks) held[i] = load_chunk<WHOLE>(a, x, tid + 256 * i);   // (zeros past the last)
  u16x2 tops2 = {0, 0};
#pragma unroll
  for (int i = 0; i < kHeld; ++i) tops2 = largest_of(held[i], tops2);
  for (int c = tid + 256 * kHeld; c < chunks; c += 256) tops2 = largest_of(load_chunk<WHOLE>(a, x, c), tops2);
  uint32_t top = wave_largest(tops2);
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = top > tops[w] ? top : tops[w];
  const RowScale rs = row_scale<BF16>(top);
  if (tid == 0) a.scale[row] = rs.scale;
  int64_t tile = row >> 4;
  int r = (int)(row & 15);
  if (a.channels) {
    tile = 2 * (row >> 5) + (row >> 2 & 1);
    r = (int)(4 * (row >> 3 & 3) + (row & 3));
  }
  uint8_t* out = a.tiles + tile * 16 * a.Kp + r * 16;
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (tid + 256 * i < chunks) {
      const int c = tid + 256 * i;
      *(u32x4*)(out + (int64_t)(c >> 2) * kTile + (c & 3) * 256) = codes_of<BF16>(held[i], rs);
    }
  for (int c = tid + 256 * kHeld; c < chunks; c += 256)
    *(u32x4*)(out + (int64_t)(c >> 2) * kTile + (c & 3) * 256) = codes_of<BF16>(load_chunk<WHOLE>(a, x, c), rs);
}

// ---------------------------------------------------------------- the product
struct ProductArgs {
  const uint8_t *x, *w;          // tiles
  const float *xs, *ws;          // scales of rows and channels
  void* y;
  int64_t ys, M, N;
  int32_t MT, NT, KT;            // tiles of rows, channels and inputs (even)
  int32_t splits;                // of the inputs among workgroups
  uint32_t* tickets;             // a word for each block of outputs, 0
  uint64_t* parts;               // its splits' sums
  uint32_t row_blocks, channel_blocks;   // of large tiles
  uint32_t whole;                // workgroups with a large tile; the others have parts of one
};

// Eight sums of a row and eight channels, scaled and stored.  The scales'
// product first: it is the same in either order, and while it is a normal
// number of binary32 the result is within three roundings of the formula.  Held as binary32
// before it is rounded to the output's type, in every kernel alike.
struct Row8 { int v[8]; };
template <int DTYPE, bool WIDE>
__device__ __forceinline__ void store_row8(__amdgpu_buffer_rsrc_t rsrc, uint32_t at, int valid, const Row8& sum,
                                           float token, const float* channel) {
  float v[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    v[r] = (float)sum.v[r] * (token * channel[r]);
    asm("" : "+v"(v[r]));
  }
  constexpr uint32_t kOutside = 0x80000000u;   // past every resource: not stored
  if constexpr (DTYPE == 2) {
    u32x4 o[2];
#pragma unroll
    for (int r = 0; r < 8; ++r) o[r >> 2][r & 3] = __builtin_bit_cast(uint32_t, v[r]);
    if constexpr (WIDE) {
      const uint32_t cell = valid > 0 ? at : kOutside;
      __builtin_amdgcn_raw_buffer_store_b128(o[0], rsrc, cell, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(o[1], rsrc, cell + 16, 0, 0);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(o[r >> 2][r & 3], rsrc, r < valid ? at + 4 * r : kOutside, 0, 0);
    }
  } else {
    u16x8 o;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (DTYPE == 0) o[r] = f2h(v[r]);
      else o[r] = __builtin_bit_cast(uint16_t, (__bf16)v[r]);
    }
    if constexpr (WIDE) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), rsrc, valid > 0 ? at : kOutside, 0, 0);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        __builtin_amdgcn_raw_buffer_store_b16(o[r], rsrc, r < valid ? at + 2 * r : kOutside, 0, 0);
    }
  }
}

// Rows m0 ... + 15 of y from channel n0 on, as far as there are any.  (16 rows of
// at most 2^25 values stay below 2^31 bytes.)
template <int DTYPE>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of_y(const ProductArgs& a, int64_t m0, int64_t n0) {
  constexpr int kSize = DTYPE == 2 ? 4 : 2;
  const int64_t rows = a.M - m0 < 16 ? a.M - m0 : 16;
  const int64_t bytes = rows > 0 && n0 < a.N ? ((rows - 1) * a.ys + a.N - n0) * kSize : 0;
  return __builtin_amdgcn_make_buffer_rsrc((uint8_t*)a.y + (bytes ? (m0 * a.ys + n0) * kSize : 0), 0, (int)bytes,
                                           0x00027000);
}

// Sums of splits meet in memory that all XCDs see at one place (stores and
// loads that are not kept in an XCD's L2), the workgroup that comes last adds
// them: whole numbers, so the order does not matter.
__device__ __forceinline__ void put(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether the workgroup is the last of its block's splits.  Its stores have
// completed: each wave waits for its own before the barrier.
__device__ __forceinline__ bool comes_last(const ProductArgs& a, uint32_t block, uint32_t* shared) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    *shared = __hip_atomic_fetch_add(a.tickets + block, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return *shared == (uint32_t)a.splits - 1;
}

__device__ __forceinline__ void tile_to_lds(const uint8_t* tile, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(tile),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void meet() { asm volatile("s_barrier" ::: "memory"); }

// A block of 16 BM rows by 16 BN channels over input tiles k0 ... k1 - 1 by
// WM x WN waves.  The operands of STAGES stages of KS input tiles lie in LDS,
// brought by direct transfers STAGES - 1 ahead; a wave reads the next tile's
// operands while the matrix cores have this one's, and meets the others once a
// stage.
// A large block's input tile is 1,024 clocks of products a SIMD and 128 KB of LDS
// traffic, about as many clocks; alone it takes 1,250, with all CUs at it up to
// 1,700 (a tenth of that are operands that miss the L2).  8,192 cubed: 410 us, 2.7
// POP/s (450 with the codes' launch).  Four waves with 128 x 128 outputs each (a quarter less LDS traffic, one
// wave a SIMD), five stages, wave priorities and all reads in front of the
// products were not faster; the stores at the end are 5 us a block.  In the block
// of 128 x 128, two groups of four waves with every other input tile each (a
// quarter less LDS traffic) gained 3% and were left out.
template <int DTYPE, bool WIDE, int BM, int BN, int WM, int WN, int STAGES, int KS, bool SPLIT = false>
__device__ __forceinline__ void tile_block(const ProductArgs& a, uint8_t* lds, int m0, int n0, int k0, int k1, int split,
                                           uint32_t block, uint32_t* shared) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, ALL = BM + BN, L = ALL / NW;
  static_assert(ALL % NW == 0 && TN % 2 == 0 && (KS == 1 || KS == 2) && STAGES > 2, "");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const uint8_t* src[L];      // tiles past the last read the last, for outputs that are not stored
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int t = wave * L + j;
    const bool weights = t < BN;
    int64_t tile = weights ? n0 + t : m0 + t - BN;
    const int64_t most = (weights ? a.NT : a.MT) - 1;
    tile = tile < most ? tile : most;
    src[j] = (weights ? a.w : a.x) + (tile * a.KT + k0) * kTile;
  }
  const uint32_t base = lds_address(lds) + wave * L * kTile, off = lane * 16;
  auto issue = [&](int stage) {
#pragma unroll
    for (int j = 0; j < L; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k) tile_to_lds(src[j] + k * kTile, off, base + ((stage * KS + k) * ALL + j) * kTile);
  };
  int issued = k0;
  auto advance = [&]() {      // past the end the last stage again, which nobody reads
    issued += KS;
    const int step = issued < k1 ? KS * kTile : 0;
#pragma unroll
    for (int j = 0; j < L; ++j) src[j] += step;
  };
  i32x4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  i32x4 wf[2][TN], xf[2][TM];
  auto fetch = [&](int slot, int step) {
    const uint8_t* s = lds + step * ALL * kTile + off;
#pragma unroll
    for (int i = 0; i < TN; ++i) wf[slot][i] = *(const i32x4*)(s + (wn * TN + i) * kTile);
#pragma unroll
    for (int j = 0; j < TM; ++j) xf[slot][j] = *(const i32x4*)(s + (BN + wm * TM + j) * kTile);
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    issue(s);
    advance();
  }
  wait_loads<(STAGES - 2) * L * KS>();
  meet();
  fetch(0, 0);
  int write = STAGES - 1, read = 1;
  for (int kt = k0; kt < k1; kt += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      __builtin_amdgcn_sched_barrier(0);
      if (KS == 1 || u == 1) {
        // the next stage is here, and nobody reads the one before this any more
        wait_loads<(STAGES - 3) * L * KS>();
        meet();
        issue(write);
        advance();
        write = write + 1 < STAGES ? write + 1 : 0;
      }
      __builtin_amdgcn_sched_barrier(0);
      fetch(1 - u, read);
      read = read + 1 < STAGES * KS ? read + 1 : 0;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i], xf[u][j], acc[i][j], 0, 0, 0);
      // reads between the products, not in front of them
      constexpr int PER = TN * TM / (TN + TM);
#pragma unroll
      for (int q = 0; q < TN + TM; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, TN * TM - PER * (TN + TM), 0);
    }
  }
  if (SPLIT && a.splits > 1) {
    constexpr int kPart = NW * TN * TM * 128;   // 8-byte words of a block's sums
    uint64_t* mine = a.parts + ((int64_t)block * a.splits) * kPart + wave * TN * TM * 128 + lane;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          put(mine + (int64_t)split * kPart + ((i * TM + j) * 2 + h) * 64,
              (uint64_t)(uint32_t)acc[i][j][2 * h] | (uint64_t)(uint32_t)acc[i][j][2 * h + 1] << 32);
    if (!comes_last(a, block, shared)) return;
    // three splits' sums on their way at a time (one after the other each costs its way through memory)
    constexpr int kAtOnce = 3, kWords = TN * TM * 2;
    for (int s = 1; s < a.splits; s += kAtOnce) {
      uint64_t v[kAtOnce][kWords];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int other = split + s + q, from = other < a.splits ? other : other - a.splits;
        if (s + q < a.splits) {
#pragma unroll
          for (int e = 0; e < kWords; ++e) v[q][e] = get(mine + (int64_t)from * kPart + e * 64);
        }
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
        if (s + q < a.splits) {
#pragma unroll
          for (int e = 0; e < kWords; ++e) {
            acc[e / 2 / TM][e / 2 % TM][2 * (e & 1)] += (int)(uint32_t)v[q][e];
            acc[e / 2 / TM][e / 2 % TM][2 * (e & 1) + 1] += (int)(uint32_t)(v[q][e] >> 32);
          }
        }
    }
  }
  // every scale of the wave's block in one go, then its outputs
  float ts[TM], cs[TN / 2][8];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int64_t m = (int64_t)(m0 + wm * TM + j) * 16 + (lane & 15);
    ts[j] = a.xs[m < a.M ? m : a.M - 1];
  }
  const int64_t first = (int64_t)(n0 + wn * TN) * 16 + 8 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < TN / 2; ++i)
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t n = first + 32 * i + r;
      cs[i][r] = a.ws[n < a.N ? n : a.N - 1];
    }
  wait_loads<0>();            // the transfers that nobody read, too
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const __amdgpu_buffer_rsrc_t y = rows_of_y<DTYPE>(a, (int64_t)(m0 + wm * TM + j) * 16, (int64_t)(n0 + wn * TN) * 16);
#pragma unroll
    for (int i = 0; i < TN / 2; ++i) {
      Row8 s;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s.v[r] = acc[2 * i][j][r];
        s.v[r + 4] = acc[2 * i + 1][j][r];
      }
      const int64_t left = a.N - (first + 32 * i);
      const uint32_t at = (uint32_t)(((lane & 15) * a.ys + 32 * i + 8 * (lane >> 4)) * (DTYPE == 2 ? 4 : 2));
      store_row8<DTYPE, WIDE>(y, at, left < 8 ? (int)left : 8, s, ts[j], cs[i]);
    }
  }
}

// Workgroups take consecutive blocks within an XCD, eight row blocks before the
// next channel block, so that the 32 of an XCD share operands in its L2.
__device__ __forceinline__ void block_place(uint32_t linear, uint32_t rows, uint32_t channels, uint32_t& rb, uint32_t& cb) {
  const uint32_t group = linear / (8 * channels), in = linear - group * 8 * channels;
  const uint32_t here = rows - group * 8 < 8 ? rows - group * 8 : 8;
  rb = group * 8 + in % here;
  cb = in / here;
}
__device__ __forceinline__ uint32_t on_one_xcd(uint32_t index, uint32_t count) {
  const uint32_t per = count >> 3, more = count & 7, xcd = index & 7;
  return xcd * per + (xcd < more ? xcd : more) + (index >> 3);
}

constexpr int kBig = 16;      // tiles a side of a large block
constexpr int kTileLds = 128 * 1024;

// PART: what the workgroups past `whole` take.  0: there are none; 1: halves of a
// large block's channels; 2: its quarters; 3: blocks of a quarter's size, of
// which row_blocks and channel_blocks then count, and splits of their inputs.
template <int DTYPE, bool WIDE, int PART>
__global__ __launch_bounds__(512, 2) void k_int8_tiles(ProductArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint32_t* shared = (uint32_t*)(lds + kTileLds);
  const uint32_t blocks = a.row_blocks * a.channel_blocks;
  uint32_t rb, cb;
  if constexpr (PART == 3) {
    const uint32_t index = on_one_xcd(blockIdx.x, blocks * a.splits), block = index / a.splits,
                   split = index - block * a.splits;
    block_place(block, a.row_blocks, a.channel_blocks, rb, cb);
    const int pairs = a.KT / 2;
    const int k0 = 2 * (int)((int64_t)pairs * split / a.splits), k1 = 2 * (int)((int64_t)pairs * (split + 1) / a.splits);
    tile_block<DTYPE, WIDE, 8, 8, 4, 2, 4, 2, true>(a, lds, rb * 8, cb * 8, k0, k1, split, block, shared);
    return;
  }
  if (blockIdx.x < a.whole) {
    block_place(on_one_xcd(blockIdx.x, a.whole), a.row_blocks, a.channel_blocks, rb, cb);
    tile_block<DTYPE, WIDE, kBig, kBig, 4, 2, 4, 1>(a, lds, rb * kBig, cb * kBig, 0, a.KT, 0, 0, shared);
  } else if constexpr (PART == 1 || PART == 2) {
    const uint32_t index = on_one_xcd(blockIdx.x - a.whole, (blocks - a.whole) * 2 * PART);
    block_place(a.whole + index / (2 * PART), a.row_blocks, a.channel_blocks, rb, cb);
    const int m0 = rb * kBig + (PART == 2 && (index & 2) ? 8 : 0), n0 = cb * kBig + (index & 1) * 8;
    if (m0 >= a.MT || n0 >= a.NT) return;
    if constexpr (PART == 1) tile_block<DTYPE, WIDE, kBig, 8, 4, 2, 4, 1>(a, lds, m0, n0, 0, a.KT, 0, 0, shared);
    else tile_block<DTYPE, WIDE, 8, 8, 4, 2, 4, 2>(a, lds, m0, n0, 0, a.KT, 0, 0, shared);
  }
}

// A few rows: bound by the weights' bytes.  A workgroup takes 16 TILES channels,
// its waves a range of inputs each; operands go straight to registers, DEEP
// input tiles ahead.  FUSED rows at most (0: the
// codes are there): the workgroup forms the rows' codes itself, in LDS, while
// its first weights are on their way.
template <int DTYPE, bool WIDE, int BM, int TILES, int WAVES, int DEEP, int FUSED, bool BF16, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, WAVES <= 8 ? 2 : 4) void k_int8_few(ProductArgs a, RowArgs ra) {
  static_assert(BM == 1 || !FUSED, "");
  __shared__ i32x4 sums[WAVES][TILES * BM][64];
  __shared__ uint32_t shared;
  __shared__ uint32_t tops[FUSED ? FUSED : 1][WAVES];
  __shared__ __attribute__((aligned(16))) uint8_t codes[FUSED ? FUSED * kFusedInputs : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t group = SPLIT ? blockIdx.x / a.splits : blockIdx.x, split = SPLIT ? blockIdx.x - group * a.splits : 0;
  const int pieces = SPLIT ? a.splits * WAVES : WAVES, piece = split * WAVES + wave;
  const int k0 = a.KT * piece / pieces, n = a.KT * (piece + 1) / pieces - k0;
  const uint8_t *wp[TILES], *xp[BM];
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    const int64_t t = (int64_t)TILES * group + i < a.NT ? (int64_t)TILES * group + i : a.NT - 1;
    wp[i] = a.w + (t * a.KT + k0) * kTile;
  }
#pragma unroll
  for (int j = 0; j < BM; ++j) xp[j] = a.x + ((int64_t)(j < a.MT ? j : a.MT - 1) * a.KT + k0) * kTile;
  i32x4 acc[TILES][BM];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int j = 0; j < BM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  i32x4 wf[DEEP][TILES], xf[DEEP][BM];
  auto load = [&](int slot, int k) {
    const int at = (k < n ? k : n - 1) * kTile + lane * 16;
#pragma unroll
    for (int i = 0; i < TILES; ++i) wf[slot][i] = *(const i32x4*)(wp[i] + at);
    if constexpr (!FUSED) {
#pragma unroll
      for (int j = 0; j < BM; ++j) xf[slot][j] = *(const i32x4*)(xp[j] + at);
    }
  };
  if (n > 0) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) load(d, d);
  }
  float token = 0.f;      // the scale of row lane % 16
  if constexpr (FUSED) {
    constexpr int THREADS = 64 * WAVES, HELD = (kFusedInputs / 16 + THREADS - 1) / THREADS;
    const int chunks = (int)(ra.Kp / 16);
    Chunk held[FUSED][HELD];
#pragma unroll
    for (int r = 0; r < FUSED; ++r) {
      const uint16_t* x = ra.x + (r < ra.rows ? r : ra.rows - 1) * ra.stride;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        if (THREADS * i >= chunks) held[r][i] = Chunk{};
        else held[r][i] = load_chunk<true>(ra, x, tid + THREADS * i);
      }
    }
#pragma unroll
    for (int r = 0; r < FUSED; ++r) {
      u16x2 pair = {0, 0};
#pragma unroll
      for (int i = 0; i < HELD; ++i) pair = largest_of(held[r][i], pair);
      const uint32_t top = wave_largest(pair);
      if (lane == 0) tops[r][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < FUSED; ++r) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) t = t > tops[r][w] ? t : tops[r][w];
      const RowScale rs = row_scale<BF16>(t);
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (tid + THREADS * i < chunks)
          *(u32x4*)(codes + r * kFusedInputs + 16 * (tid + THREADS * i)) = codes_of<BF16>(held[r][i], rs);
      if ((lane & 15) == r) token = rs.scale;
    }
    __syncthreads();
  }
  const uint8_t* mine16 = codes + (FUSED ? (lane & (FUSED - 1)) * kFusedInputs : 0) + k0 * 64 + 16 * (lane >> 4);
  auto multiply = [&](int slot, int k) {
    if constexpr (FUSED) xf[slot][0] = *(const i32x4*)(mine16 + k * 64);
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int j = 0; j < BM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[slot][i], xf[slot][j], acc[i][j], 0, 0, 0);
  };
  constexpr int kBurst = 2;            // tiles whose loads go together
  int k = 0;
  for (; k + DEEP <= n; k += DEEP) {   // (without a branch inside, so that a wait is for one tile's loads)
#pragma unroll
    for (int d = 0; d < DEEP; d += kBurst) {
#pragma unroll
      for (int e = 0; e < kBurst; ++e) multiply(d + e, k + d + e);
#pragma unroll
      for (int e = 0; e < kBurst; ++e) load(d + e, k + d + e + DEEP);
      __builtin_amdgcn_sched_barrier(0);   // (left alone, the scheduler sinks loads to their use)
    }
  }
#pragma unroll
  for (int d = 0; d < DEEP; ++d)
    if (k + d < n) multiply(d, k + d);
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int j = 0; j < BM; ++j) sums[wave][i * BM + j][lane] = acc[i][j];
  __syncthreads();
  // 32 channels of 16 rows a wave at a time
  constexpr int kAll = TILES / 2 * BM, kUnits = (kAll + WAVES - 1) / WAVES;
  Row8 total[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = wave + u * WAVES, i = unit % (TILES / 2), j = unit / (TILES / 2);
    if (unit >= kAll) break;
    i32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      lo += sums[w][2 * i * BM + j][lane];
      hi += sums[w][(2 * i + 1) * BM + j][lane];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      total[u].v[r] = lo[r];
      total[u].v[r + 4] = hi[r];
    }
  }
  if (SPLIT && a.splits > 1) {
    constexpr int kPart = kAll * 256;
    uint64_t* mine = a.parts + (int64_t)group * a.splits * kPart + lane;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = wave + u * WAVES;
      if (unit >= kAll) break;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        put(mine + (int64_t)split * kPart + (unit * 4 + h) * 64,
            (uint64_t)(uint32_t)total[u].v[2 * h] | (uint64_t)(uint32_t)total[u].v[2 * h + 1] << 32);
    }
    if (!comes_last(a, group, &shared)) return;
    for (uint32_t s = 0; s < (uint32_t)a.splits; ++s) {
      if (s == split) continue;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int unit = wave + u * WAVES;
        if (unit >= kAll) break;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint64_t v = get(mine + (int64_t)s * kPart + (unit * 4 + h) * 64);
          total[u].v[2 * h] += (int)(uint32_t)v;
          total[u].v[2 * h + 1] += (int)(uint32_t)(v >> 32);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = wave + u * WAVES, i = unit % (TILES / 2), j = unit / (TILES / 2);
    if (unit >= kAll) break;
    const int64_t m = 16 * j + (lane & 15), n0 = (int64_t)group * (16 * TILES) + 32 * i, first = n0 + 8 * (lane >> 4);
    float cs[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) cs[r] = a.ws[first + r < a.N ? first + r : a.N - 1];
    if constexpr (!FUSED) token = a.xs[m < a.M ? m : a.M - 1];
    const int64_t left = a.N - first;
    const int valid = left < 8 ? (int)left : 8;
    const uint32_t at = (uint32_t)(((lane & 15) * a.ys + 8 * (lane >> 4)) * (DTYPE == 2 ? 4 : 2));
    const __amdgpu_buffer_rsrc_t y = rows_of_y<DTYPE>(a, 16 * j, n0);
    store_row8<DTYPE, WIDE>(y, at, valid, total[u], token, cs);
  }
}

// ---------------------------------------------------------------- which kernel
// Rows up to which k_int8_few is taken: 32 rows, 4,096 -> 18,560 20 us, 64 rows 24
// and 21 in blocks of 128 x 128, 65 rows 30 and 20, 128 rows 33 and 21: for so many
// channels the border could lie somewhat lower.  Where these blocks are few, twice
// the rows: 128 rows, 8,192 -> 4,096 17.5 us against 20.6 with the inputs of 32
// blocks split in four.
constexpr int64_t kFewRows = 64;

struct Plan {
  int few;                 // row tiles of k_int8_few, or 0
  int fused;               // rows whose codes it forms itself, at most
  int shape;               // of its workgroups: 0 64 channels and 4 waves, 1 32 and 4, 2 32 and 16 with splits
  int part;                // how blocks past `whole` are cut
  int splits;
  uint32_t rb, cb, whole, grid;
  int64_t tickets, parts;  // words of 4 and of 8 bytes
};

static Plan int8_plan(int64_t M, int64_t N, int64_t K, bool whole) {
  Plan p{};
  const int64_t MT = row_tiles(M), NT = channel_tiles(N), KT = padded_inputs(K) / 64;
  p.splits = 1;
  const int64_t pairs = NT / 2;
  if (M <= kFewRows || (M <= 2 * kFewRows && pairs < 256)) {
    p.few = MT == 1 ? 1 : (MT == 2 ? 2 : (MT <= 4 ? 4 : 8));
    if (M <= 4 && K <= kFusedInputs && whole) p.fused = M <= 2 ? (int)M : 4;
    // us by shape 0 / 1 / 2: 24 rows, 4,096 -> 256,000 200 / 220 / 275; 32 rows, 4,096 -> 18,560 23 / 20 / 23; 16 rows,
    // 8,192 -> 4,096 14.0 / 12.5 / 12.4, 64 rows 18.1 / 16.7 / 14.6
    p.shape = p.fused ? 1 : (pairs < 256 ? 2 : (pairs < 2048 ? 1 : 0));
    p.grid = (uint32_t)(p.shape ? pairs : (NT + 3) / 4);
    if (p.shape == 2) {
      int64_t s = 256 / pairs, most = KT / 64;
      s = s < most ? s : most;
      p.splits = (int)(s < 1 ? 1 : s < 8 ? s : 8);
      p.grid *= p.splits;
      if (p.splits > 1) {
        p.tickets = pairs;
        p.parts = pairs * p.splits * p.few * 256;
      }
    }
    return p;
  }
  const int64_t rb = (MT + kBig - 1) / kBig, cb = (NT + kBig - 1) / kBig, all = rb * cb, rest = all % 256;
  const int64_t rs = (MT + 7) / 8, cs = (NT + 7) / 8, small = rs * cs;
  // Rounds of 256 workgroups, in large blocks: the last round's blocks whole, in
  // halves, in quarters, or everything in blocks of a quarter's size.  A round of
  // 4,096 inputs takes 45 us, 31 in halves, 19 in quarters (68, 43 and 30 with the
  // codes' launch and the call's start and end).  2,048 rows, 4,096 -> 18,560: 164 us
  // whole, 151 with the last 72 of 584 in halves, 155 in quarters; 512 rows 51 whole,
  // 61 in halves or quarters.
  const double full = (double)(all / 256), rounds[4] = {full + (rest ? 1 : 0), full + 0.62 * ((2 * rest + 255) / 256),
                                                        full + 0.42 * ((4 * rest + 255) / 256),
                                                        0.42 * ((small + 255) / 256)};
  for (int i = 1; i < 4; ++i)
    if (rounds[i] < rounds[p.part]) p.part = i;
  if (2 * small <= 256) p.part = 3;       // and split inputs: 192 rows, 8,192 -> 4,096 32 us unsplit, 23 in four
  p.rb = (uint32_t)(p.part == 3 ? rs : rb);
  p.cb = (uint32_t)(p.part == 3 ? cs : cb);
  p.whole = (uint32_t)(p.part == 0 ? all : (p.part == 3 ? 0 : all - rest));
  if (p.part == 3) {
    int64_t s = 256 / small;
    const int64_t most = KT / 32;
    s = s < most ? s : most;
    p.splits = (int)(s < 1 ? 1 : (s < 8 ? s : 8));
    if (p.splits > 1) {
      p.tickets = small;
      p.parts = small * p.splits * 8192;
    }
    p.grid = (uint32_t)(small * p.splits);
  } else p.grid = (uint32_t)(p.whole + 2 * p.part * (all - p.whole));
  return p;
}

template <int DTYPE, bool WIDE, int PART>
static int tiles_launch(const Plan& p, const ProductArgs& a, hipStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  if (int rc = m2r_allow_lds((const void*)k_int8_tiles<DTYPE, WIDE, PART>, kTileLds + 16, allowed)) return rc;
  hipLaunchKernelGGL((k_int8_tiles<DTYPE, WIDE, PART>), dim3(p.grid), dim3(512), kTileLds + 16, stream, a);
  return 0;
}
template <int DTYPE, bool WIDE, int BM, int TILES, int WAVES, int DEEP, int FUSED = 0, bool BF16 = false, bool SPLIT = false>
static void few_launch(const Plan& p, const ProductArgs& a, const RowArgs& r, hipStream_t stream) {
  hipLaunchKernelGGL((k_int8_few<DTYPE, WIDE, BM, TILES, WAVES, DEEP, FUSED, BF16, SPLIT>), dim3(p.grid), dim3(64 * WAVES), 0, stream, a,
                     r);
}
template <int DTYPE, bool WIDE>
static void few(const Plan& p, const ProductArgs& a, const RowArgs& r, bool bf16, hipStream_t stream) {
  if (p.fused == 1) bf16 ? few_launch<DTYPE, WIDE, 1, 2, 4, 8, 1, true>(p, a, r, stream) : few_launch<DTYPE, WIDE, 1, 2, 4, 8, 1>(p, a, r, stream);
  else if (p.fused == 2) bf16 ? few_launch<DTYPE, WIDE, 1, 2, 4, 8, 2, true>(p, a, r, stream) : few_launch<DTYPE, WIDE, 1, 2, 4, 8, 2>(p, a, r, stream);
  else if (p.fused == 4) bf16 ? few_launch<DTYPE, WIDE, 1, 2, 4, 8, 4, true>(p, a, r, stream) : few_launch<DTYPE, WIDE, 1, 2, 4, 8, 4>(p, a, r, stream);
  else if (p.shape == 0) {
    if (p.few == 1) few_launch<DTYPE, WIDE, 1, 4, 4, 4>(p, a, r, stream);
    else if (p.few == 2) few_launch<DTYPE, WIDE, 2, 4, 4, 4>(p, a, r, stream);
    else few_launch<DTYPE, WIDE, 4, 4, 4, 4>(p, a, r, stream);
  } else if (p.shape == 1) {
    if (p.few == 1) few_launch<DTYPE, WIDE, 1, 2, 4, 8>(p, a, r, stream);
    else if (p.few == 2) few_launch<DTYPE, WIDE, 2, 2, 4, 8>(p, a, r, stream);
    else few_launch<DTYPE, WIDE, 4, 2, 4, 8>(p, a, r, stream);
  } else {
    if (p.few == 1) few_launch<DTYPE, WIDE, 1, 2, 16, 4, 0, false, true>(p, a, r, stream);
    else if (p.few == 2) few_launch<DTYPE, WIDE, 2, 2, 16, 4, 0, false, true>(p, a, r, stream);
    else if (p.few == 4) few_launch<DTYPE, WIDE, 4, 2, 16, 2, 0, false, true>(p, a, r, stream);
    else few_launch<DTYPE, WIDE, 8, 2, 8, 2, 0, false, true>(p, a, r, stream);
  }
}
template <int DTYPE, bool WIDE>
static int int8_product(const Plan& p, const ProductArgs& a, const RowArgs& r, bool bf16, hipStream_t stream) {
  if (p.few) few<DTYPE, WIDE>(p, a, r, bf16, stream);
  else {
    int rc;
    if (p.part == 0) rc = tiles_launch<DTYPE, WIDE, 0>(p, a, stream);
    else if (p.part == 1) rc = tiles_launch<DTYPE, WIDE, 1>(p, a, stream);
    else if (p.part == 2) rc = tiles_launch<DTYPE, WIDE, 2>(p, a, stream);
    else rc = tiles_launch<DTYPE, WIDE, 3>(p, a, stream);
    if (rc) return rc;
  }
  return m2r_check(hipGetLastError(), "int8 product launch");
}

}  // namespace m2r

using namespace m2r;

static int int8_rows(const RowArgs& a, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)((a.rows + 127) / 128 * 128)), block(256);
  auto k = dtype == 0 ? (a.whole ? k_int8_rows<false, true> : k_int8_rows<false, false>)
                      : (a.whole ? k_int8_rows<true, true> : k_int8_rows<true, false>);
  hipLaunchKernelGGL(k, grid, block, 0, stream, a);
  return m2r_check(hipGetLastError(), "int8 rows launch");
}

// Rows of whole sixteens at 16-byte boundaries.
static bool whole_rows(const void* x, int64_t stride, int64_t K) {
  return !((uintptr_t)x & 15) && !(stride & 7) && !(K & 15);
}

// (k_int8_rows has 256 threads a row and whole 128s of rows.)
static int int8_limits(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0) return m2r_fail("int8: non-positive shape");
  if (!m2r_grid_fits((rows + 127) / 128 * 128, 256) || K > 131072) return m2r_fail("int8: size limits");
  return 0;
}

extern "C" int64_t m2r_int8_weight_bytes(int64_t N, int64_t K) {
  if (N <= 0 || K <= 0) return 0;
  return channel_tiles(N) * 16 * padded_inputs(K);
}

extern "C" int m2r_int8_quantize(const void* w, int dtype, int64_t w_stride, void* tiles, float* scale, int64_t N,
                                 int64_t K, hipStream_t stream) {
  if (int rc = int8_limits(N, K)) return rc;
  if (dtype < 0 || dtype > 1) return m2r_fail("int8: weights must be binary16 or bfloat16");
  if (!w || !tiles || !scale) return m2r_fail("int8: null pointer");
  if (w_stride < 0) return m2r_fail("int8: negative stride");
  if ((uintptr_t)tiles & 15) return m2r_fail("int8: tiles must be 16-byte aligned");
  const RowArgs r{(const uint16_t*)w, w_stride, N, K, padded_inputs(K), (uint8_t*)tiles, scale, nullptr, 0, 1,
                  (int)whole_rows(w, w_stride, K)};
  return int8_rows(r, dtype, stream);
}

// Codes, scales, then the tickets and sums of splits, each from 256 bytes on.
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
static int64_t int8_codes_bytes(int64_t M, int64_t K) { return up256(row_tiles(M) * 16 * padded_inputs(K)); }

extern "C" int64_t m2r_int8_linear_workspace(const void* x, int64_t x_stride, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = int8_plan(M, N, K, whole_rows(x, x_stride, K));
  if (p.fused) return 0;
  return int8_codes_bytes(M, K) + up256(4 * M) + up256(4 * p.tickets) + 8 * p.parts;
}

extern "C" int m2r_int8_linear(const void* x, int x_dtype, int64_t x_stride, const void* w_tiles, const float* w_scale,
                               void* y, int y_dtype, int64_t y_stride, int64_t M, int64_t N, int64_t K, void* workspace,
                               int64_t workspace_bytes, hipStream_t stream) {
  if (N <= 0) return m2r_fail("int8: non-positive shape");
  if (int rc = int8_limits(M, K)) return rc;
  if (N > (int64_t)1 << 24 || y_stride > (int64_t)1 << 25) return m2r_fail("int8: size limits");
  if (x_dtype < 0 || x_dtype > 1) return m2r_fail("int8: x must be binary16 or bfloat16");
  if (y_dtype < 0 || y_dtype > 2) return m2r_fail("int8: y must be binary16, bfloat16 or binary32");
  for (const void* p : {x, w_tiles, (const void*)w_scale, (const void*)y})
    if (!p) return m2r_fail("int8: null pointer");
  if (x_stride < 0) return m2r_fail("int8: negative stride");
  if (y_stride < N) return m2r_fail("int8: rows overlap");
  if ((uintptr_t)w_tiles & 15) return m2r_fail("int8: tiles must be 16-byte aligned");
  const int64_t needed = m2r_int8_linear_workspace(x, x_stride, M, N, K);
  if (needed && (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < needed))
    return m2r_fail("int8: workspace too small or not 16-byte aligned");
  const int64_t MT = row_tiles(M), NT = channel_tiles(N);
  if ((MT + kBig - 1) / kBig * ((NT + kBig - 1) / kBig) > 0x7fffffff / 64) return m2r_fail("int8: grid limits exceeded");
  // wide: whole eights of channels, dword-aligned, stored by 16 bytes
  const bool whole = whole_rows(x, x_stride, K), wide = !(N & 7) && !(y_stride & 1) && !((uintptr_t)y & 3);
  const Plan p = int8_plan(M, N, K, whole);
  if (!p.few && !m2r_grid_fits(p.grid, 512)) return m2r_fail("int8: grid limits exceeded");
  uint8_t* codes = (uint8_t*)workspace;
  float* scale = (float*)(codes + int8_codes_bytes(M, K));
  uint32_t* tickets = (uint32_t*)((uint8_t*)scale + up256(4 * M));
  uint64_t* parts = (uint64_t*)((uint8_t*)tickets + up256(4 * p.tickets));
  const RowArgs r{(const uint16_t*)x, x_stride, M, K, padded_inputs(K), codes, scale, tickets, p.tickets, 0, (int)whole};
  if (!p.fused)
    if (int rc = int8_rows(r, x_dtype, stream)) return rc;
  const ProductArgs a{codes, (const uint8_t*)w_tiles, scale, w_scale, y, y_stride, M, N, (int32_t)MT, (int32_t)NT,
                      (int32_t)(padded_inputs(K) / 64), p.splits, tickets, parts, p.rb, p.cb, p.whole};
  if (y_dtype == 0)
    return wide ? int8_product<0, true>(p, a, r, x_dtype, stream) : int8_product<0, false>(p, a, r, x_dtype, stream);
  if (y_dtype == 1)
    return wide ? int8_product<1, true>(p, a, r, x_dtype, stream) : int8_product<1, false>(p, a, r, x_dtype, stream);
  return wide ? int8_product<2, true>(p, a, r, x_dtype, stream) : int8_product<2, false>(p, a, r, x_dtype, stream);
}
