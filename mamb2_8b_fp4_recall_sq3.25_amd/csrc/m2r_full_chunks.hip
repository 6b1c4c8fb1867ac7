// Scan with a full-precision carry over many tokens, on the matrix cores: the
// recurrence of m2r_full.hip in chunks of 64 tokens.  With l_t the running sum
// of A dt inside a chunk, S the carry before it and S' the carry after it,
//   y_t = sum_{s <= t} (C_t . B_s) exp(l_t - l_s) dt_s x_s + exp(l_t) S C_t + D x_t
//   S'  = exp(l_63) S + sum_s exp(l_63 - l_s) dt_s x_s (x) B_s.
// The products run on binary16 matrix instructions that sum in binary32.  B, C
// and x are binary16 already; what is not goes in as several of them, scaled by
// a power of two that keeps the largest value near the top of the range.  The
// carry and the weighted x take two, 22 bits and nothing below 2^-39 of the
// largest, with a power of two for each channel, since channels do not meet in
// any product.  The weighted scores take three, down to 2^-62: decays and inputs
// that lie far apart spread them further.  The running sums l are formed in 64
// bits, since differences of them become exponents.
//
// Work: a chunk and head of 64 costs 3 products of 64 x 64 x 128 (C B^T once for
// all heads of a group), the last two twice for the halves, and 64 x 64 weights,
// whose product with x runs three times; x, y, B, C and dt move once, the
// carry stays in registers across a segment (64 values a thread, which is why
// a workgroup is 512 threads of 256 registers).  What few rows lack in
// workgroups is made up by cutting the tokens into segments: a first pass
// forms what each adds to a zero carry (x and B only), k_full_join runs the
// carries through, and the main pass starts every segment from its own.
//
// At 128 heads of 64 in 8 groups: 8,192 tokens of one row 214 us (the profiler
// has first pass 55, join 13, main pass 165 at least), 1.5 TB/s and 201 TFLOP/s
// counted token by token; 2,048 tokens 81 us; nine rows of 62 to 901 tokens 137
// us in one pass; five short prompts 28 us.  Neither memory (64 us at 8,192
// tokens) nor the matrix cores bound it: a chunk takes a workgroup 18,400 clocks,
// of which a SIMD's vector instructions are about 10,600, the LDS 4,600 and the
// matrix instructions 5,400, and they overlap little, as both waves of a SIMD are
// at the same step.  The powers of two of each channel and the weights' third
// part are 260 of a chunk's 1,320 vector instructions and 8 us of the 214.
// Weights as two bfloat16 parts, which need no power of two, but x in two parts
// as well: 250 us.  Conversions by mixed fmas that write binary16: 237 (they
// issue at half the rate).  Before these, of 218 us, leaving parts out saved: S C
// 22, the update 40, the stores 22, the loads 25, the weights 15, the scalars 10;
// and not better were: scores formed by each wave for itself, with one barrier a
// chunk (222 us for the main kernels' 177); 16 waves of 128 registers (219 for
// 221); S C behind the barrier; waves that start their chunk's parts in another
// order.
#include "m2r_full.h"
#include "m2r_abi_util.h"

namespace m2r {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) f16x4 lds_f16x4;
typedef __attribute__((address_space(3))) s16x4v lds_s16x4;

constexpr int kChunk = 64;
// B, C and x come by direct transfers (64 lanes x 16 bytes in a row), so their
// rows in LDS are dense, and their 16-byte pieces are exchanged instead, so that
// the rows that one read touches stand on different banks: piece p of row r is
// at p ^ bc_turn(r) (16 rows x 16 bytes, or transposing 8 rows x 32 bytes) or
// p ^ x_turn(r) (rows of half the length).
constexpr int kRowB = 128, kRowX = 64;
__device__ __forceinline__ int bc_turn(int row) { return ((row & 7) << 1) | ((row >> 3) & 1); }
__device__ __forceinline__ int bc_at(int row, int n) { return row * kRowB + 8 * ((n >> 3) ^ bc_turn(row)) + (n & 7); }
__device__ __forceinline__ int x_turn(int row) { return ((row >> 1) & 3) << 1; }
__device__ __forceinline__ int x_at(int row, int col) { return row * kRowX + 8 * ((col >> 3) ^ x_turn(row)) + (col & 7); }

// What the heads' tokens need besides B, C and x.  l is the running sum of
// A dt log2(e) over the chunk, r_j its value at the last token of the 16-token
// tile j; powers are of two.
template <bool OUT>
struct ChunkScalars {
  static constexpr int kOut = OUT ? kChunk : 1;
  float lh[kOut], ll[kOut];       // l as a sum of two binary32
  float lt[kOut];                 // l - r of the tile before
  float dt[kOut];
  float ws[kOut];                 // dt 2^(r_tile - l)
  float el[kOut];                 // 2^l
  // Where the carry grows, 2^(l_63 - l) may leave binary32 while what it multiplies
  // does not: its whole powers of two are kept apart.
  alignas(16) float w[kChunk];    // dt 2^(l_63 - up - l)
  float tot, up;                  // 2^(l_63 - up), max(floor(l_63), 0)
  float dtmax, unused;            // the largest finite dt
};

// `Ahead`: chunks on their way besides the one in work.
template <bool OUT>
struct ChunkShared {
  static constexpr int kAhead = OUT ? 1 : 2, kBuffers = kAhead + 1;
  uint16_t c[OUT ? kBuffers : 1][OUT ? kChunk * kRowB : 8];
  uint16_t b[kBuffers][kChunk * kRowB];
  uint16_t x[kBuffers][4][kChunk * kRowX];
  uint32_t dt[kBuffers][4][kChunk];      // as loaded, one value a word
  f32x4 scores[OUT ? 10 : 1][64];        // (C B^T) tiles on and below the diagonal, by lane
  ChunkScalars<OUT> h[2][4];
  float gmax[8];                         // largest finite score, by wave
  float undo[OUT ? 8 : 1][OUT ? 32 : 1]; // by wave and column: the carry's value to one unit of its halves
};

struct Segments {
  int64_t tokens;     // of a segment, a multiple of kChunk
  int count;
  // For rows that go on past their first segment, [count, batch, H, P, 128]:
  // 0 the row's first carry (the pool's own is overwritten by the last segment
  // while others still start), q > 0 first what segment q - 1 adds to a zero
  // carry, then (k_full_join) the carry before segment q; and the decay over
  // segment q - 1, as a factor below 2 and a power of two.
  float* state;
  f32x2* decay;       // [count, batch, H]
  bool longest_first; // the grid's y is a row's place by length, not its number
};

// The largest over the wave.  Non-negative binary32 values order as their
// bits do, NaN above infinity.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
#define M2R_MAX_DPP(ctrl)                                                                     \
  {                                                                                          \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, true); \
    v = v > o ? v : o;                                                                       \
  }
  M2R_MAX_DPP(0xB1)
  M2R_MAX_DPP(0x4E)
  M2R_MAX_DPP(0x141)
  M2R_MAX_DPP(0x140)
#undef M2R_MAX_DPP
  const auto r = __builtin_amdgcn_permlane16_swap((int)v, (int)v, false, false);
  v = (uint32_t)r[0] > (uint32_t)r[1] ? (uint32_t)r[0] : (uint32_t)r[1];
  const auto q = __builtin_amdgcn_permlane32_swap((int)v, (int)v, false, false);
  v = (uint32_t)q[0] > (uint32_t)q[1] ? (uint32_t)q[0] : (uint32_t)q[1];
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ float wave_max(float v) {
  return __builtin_bit_cast(float, wave_max_bits(__builtin_bit_cast(uint32_t, v)));
}
// The largest over the four lanes that hold the same column (lane % 16).
__device__ __forceinline__ float column_max(float v) {
  const int iv = __builtin_bit_cast(int, v);
  const auto p = __builtin_amdgcn_permlane16_swap(iv, iv, false, false);
  v = __builtin_fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1]));
  const int jv = __builtin_bit_cast(int, v);
  const auto q = __builtin_amdgcn_permlane32_swap(jv, jv, false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, (int)q[0]), __builtin_bit_cast(float, (int)q[1]));
}
__device__ __forceinline__ float finite_or_0(float v) { return __builtin_fabsf(v) < __builtin_inff() ? v : 0.f; }
// floor(log2 v) of a positive normal v (-127 for zero and subnormals).
__device__ __forceinline__ int exponent_of(float v) { return ((__builtin_bit_cast(int, v) >> 23) & 255) - 127; }
__device__ __forceinline__ float pow2(int k) { return __builtin_ldexpf(1.0f, k); }

// v scale as the sum of two binary16, `scale` a power of two that takes the
// largest value to the exponent 13: the first carries 11 bits, the second the
// next 11 (whatever is left above 2^-25), so that a product of a binary16
// factor with both keeps 22 bits, and nothing below 2^-39 of the largest; it is
// summed in binary32 by the matrix instruction.  `scale` comes with the
// conversions: v scale - high is one mixed fma.
struct Split { f16x8 hi, lo; };
__device__ __forceinline__ Split split8(const float* v, float scale) {
  Split s;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 h = __builtin_convertvector((f32x2{v[j] * scale, v[j + 1] * scale}), f16x2);
    const f16x2 l = __builtin_convertvector(
        (f32x2{__builtin_fmaf(v[j], scale, -(float)h[0]), __builtin_fmaf(v[j + 1], scale, -(float)h[1])}), f16x2);
    s.hi[j] = h[0];
    s.hi[j + 1] = h[1];
    s.lo[j] = l[0];
    s.lo[j + 1] = l[1];
  }
  return s;
}
// v as hi + lo + least 2^-kLeast, for |v| below 2^14: the third in units of its
// own, so that nothing is left out above 2^-62 of the largest, for two sums that
// meet in binary32.
constexpr int kLeast = 24;
struct Split3 { f16x8 hi, lo, least; };
__device__ __forceinline__ Split3 split8_3(const float* v, float one) {   // one: 1, not known to the compiler
  constexpr float kUp = 1 << kLeast;
  Split3 s;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 h = __builtin_convertvector((f32x2{v[j], v[j + 1]}), f16x2);
    const float r0 = __builtin_fmaf(v[j], one, -(float)h[0]), r1 = __builtin_fmaf(v[j + 1], one, -(float)h[1]);
    const f16x2 l = __builtin_convertvector((f32x2{r0, r1}), f16x2);
    const f16x2 e = __builtin_convertvector(
        (f32x2{__builtin_fmaf(r0, one, -(float)l[0]) * kUp, __builtin_fmaf(r1, one, -(float)l[1]) * kUp}), f16x2);
    s.hi[j] = h[0];
    s.hi[j + 1] = h[1];
    s.lo[j] = l[0];
    s.lo[j + 1] = l[1];
    s.least[j] = e[0];
    s.least[j + 1] = e[1];
  }
  return s;
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Four rows by 16 columns per 16 lanes, transposed: lane i gets column i of
// the four rows.  `p`: the lane's own 8 bytes (row (lane % 16) / 4, columns
// 4 (lane % 4) ...).
__device__ __forceinline__ f16x4 read_transposed(const uint16_t* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
__device__ __forceinline__ f16x8 join(f16x4 a, f16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Up to 8 binary16 values one by one, zeros after them.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, int valid) {
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < valid) v[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  return v;
}

// Buffers of `rows` rows of `cols` binary16 at a row stride: offsets past the
// last row read zeros and write nothing, and so does kOutside.
constexpr uint32_t kOutside = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const uint16_t* p, int64_t stride, int rows, int cols) {
  const int bytes = rows > 0 && cols > 0 ? (int)(((rows - 1) * stride + cols) * 2) : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0, bytes, 0x00020000);
}

// Direct transfers of 16 bytes a lane to lds + 16 lane, or of two to a word at
// lds + 4 lane, from `off` into the buffer; zeros for offsets outside.  The
// compiler does not count them: the caller waits (wait_vmcnt).
__device__ __forceinline__ void buffer_to_lds(u32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
__device__ __forceinline__ void buffer_to_lds_u16(u32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tbuffer_load_ushort %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
__device__ __forceinline__ u32x4 rows_resource(const uint16_t* p, int64_t stride, int rows, int cols) {
  const uint64_t u = (uint64_t)p;
  const uint32_t bytes = rows > 0 && cols > 0 ? (uint32_t)(((rows - 1) * stride + cols) * 2) : 0u;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

template <int CTRL>
__device__ __forceinline__ double dpp_add64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// The value of the last of the lane's 16 (row_newbcast:15).
__device__ __forceinline__ double dpp_row_last64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x15F, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), 0x15F, 0xF, 0xF, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Inclusive sum over the wave: within rows of 16 lanes, then across them.
__device__ __forceinline__ double scan_add64(double v) {
  const int lane = threadIdx.x & 63;
  v = dpp_add64<0x111>(v);   // row_shr 1, 2, 4, 8: lanes without a source add 0
  v = dpp_add64<0x112>(v);
  v = dpp_add64<0x114>(v);
  v = dpp_add64<0x118>(v);
  const double e0 = lane64(v, 15), e1 = lane64(v, 31), e2 = lane64(v, 47);
  const double before = lane < 16 ? 0.0 : (lane < 32 ? e0 : (lane < 48 ? e0 + e1 : (e0 + e1) + e2));
  return before + v;
}

typedef uint16_t h16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t m, u32x4 v) {   // pairs of binary16
  h16x2 r = __builtin_bit_cast(h16x2, m);
#pragma unroll
  for (int j = 0; j < 4; ++j) r = __builtin_elementwise_max(r, __builtin_bit_cast(h16x2, v[j] & 0x7fff7fffu));
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t m, u32x2 v) {
  return max_magnitudes(m, u32x4{v[0], v[1], 0u, 0u});
}
// Whether a pair of binary16 magnitudes has a non-finite one.
__device__ __forceinline__ bool non_finite_half(uint32_t m) { return (m & 0xffffu) >= 0x7c00u || m >= 0x7c000000u; }
// The row of at most 64 whose token count has the given place among them,
// largest first.
__device__ __forceinline__ int64_t row_by_length(const FullArgs& a, uint32_t place) {
  const int lane = threadIdx.x & 63, rows = (int)a.batch;
  const int n = lane < rows ? (int)full_row(a, lane).len : -1;
  uint32_t before = 0;
  for (int j = 0; j < rows; ++j) {
    const int o = __builtin_amdgcn_readlane(n, j);
    before += o > n || (o == n && j < lane);
  }
  return __builtin_ctzll(__ballot(lane < rows && before == place));
}

// A workgroup steps four blocks of 64 columns (a head's channels) of one
// group, two waves each, over one segment of one batch row's tokens: four
// blocks share the loads of B and C and the scores.  OUT: readouts and the
// pool's carry; else what the segment adds to a zero carry.
// The next chunk's operands are on their way into LDS while one is in work
// (two ahead without readouts, where a chunk is shorter).
template <bool ALIGNED, bool OUT>
__global__ __launch_bounds__(512, 2) void k_full_chunks(FullArgs a, Segments sg) {
  __shared__ ChunkShared<OUT> s;
  constexpr int kAhead = ChunkShared<OUT>::kAhead, kBuffers = ChunkShared<OUT>::kBuffers;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), pair = wave >> 1, half = wave & 1;
  const int lr = lane & 15, lg = lane >> 4;
  const int hpg = (int)((uint32_t)a.H / (uint32_t)a.G), per_head = (int)((a.P + 63) / 64), blocks = (hpg * per_head + 3) / 4;
  // A group's blocks G apart, on one XCD where G is a multiple of 8: B and C come
  // into one L2 (8,192 tokens: 213 MB read for 322, in the same time).
  const int blk = (int)(blockIdx.x / (uint32_t)a.G), g = (int)(blockIdx.x - blk * (uint32_t)a.G);
  const int64_t b = OUT && sg.longest_first ? row_by_length(a, blockIdx.y) : blockIdx.y, seg = blockIdx.z;

  const FullRow fr = full_row(a, b);
  const int64_t slot = fr.slot, len = fr.len;
  const int64_t t0 = seg * sg.tokens, t1 = t0 + sg.tokens < a.L ? t0 + sg.tokens : a.L;
  const int64_t n = len < t0 ? 0 : (len < t1 ? len : t1) - t0;   // the segment's tokens
  if (!OUT && len <= t1) return;                                   // no later segment reads this one

  // this pair's head and columns (idle past the group's last block)
  const int unit = blk * 4 + pair;
  const bool live = unit < hpg * per_head;
  const int64_t h = g * hpg + (live ? unit / per_head : 0), pc = (live ? unit % per_head : 0) * 64;
  const int64_t cols = live ? (a.P - pc < 64 ? a.P - pc : 64) : 0;
  const int pw = 32 * half + lr;   // the lane's first column; the second is 16 further

  if (OUT && n < t1 - t0) {   // zeros past the length
    for (int64_t i = half * 64 + lane; i < (t1 - t0 - n) * 64; i += 128) {
      const int64_t t = t0 + n + i / 64, p = i % 64;
      if (p < cols) a.y[((b * a.L + t) * a.H + h) * a.P + pc + p] = 0;
    }
  }
  if (n == 0) return;

  const float av = a.A[h];
  const FullParam skip = full_param(a.D, a.d_f32, h), shift = full_param(a.dt_bias, a.db_f32, h);
  float bias = 0.f, dh = 0.f;
  double seg_log = 0.0;   // the segment's decay so far, as a power of two

  // the loads of a chunk: B and C two, x four 16-byte pieces a thread, dt.
  // Transfer k of a wave fills rows 32 k + 4 wave ... + 3 of B and C, rows
  // 16 k + 8 half ... + 7 of its pair's x, the lane's piece at its turned place.
  const int br = 4 * wave + (lane >> 4), bpart = (lane & 15) ^ bc_turn(br);
  const int xr = 8 * half + (lane >> 3), xpart = (lane & 7) ^ x_turn(lane >> 3);
  const uint16_t *bp = a.Bm + b * a.bs_b + t0 * a.bs_l + g * 128, *cp = a.Cm + b * a.cs_b + t0 * a.cs_l + g * 128;
  const uint16_t *xp = a.x + b * a.xs_b + t0 * a.xs_l + h * a.P + pc, *dp = a.dt + b * a.ds_b + t0 * a.ds_l + h;
  const int xcols = (int)cols - 8 * xpart;
  const uint32_t xoff = xcols > 0 ? (uint32_t)(2 * (xr * a.xs_l + 8 * xpart)) : kOutside;
  const uint32_t boff = (uint32_t)(2 * (br * a.bs_l + 8 * bpart)), coff = (uint32_t)(2 * (br * a.cs_l + 8 * bpart));
  const uint32_t doff = (uint32_t)(2 * lane * a.ds_l);
  // the wave that prepares its pair's scalars: one of the two on each SIMD
  const bool scalars = half == pair >> 1;
  auto load_chunk = [&](int64_t c0, int buf) {   // tokens t0 + c0 ...
    const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
    const uint16_t *bs = bp + c0 * a.bs_l, *cs = cp + c0 * a.cs_l, *xs = xp + c0 * a.xs_l, *ds = dp + c0 * a.ds_l;
    if constexpr (ALIGNED) {
      const u32x4 xb = rows_resource(xs, a.xs_l, left, (int)cols), bb = rows_resource(bs, a.bs_l, left, 128);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        buffer_to_lds(xb, xoff + (uint32_t)(32 * k * a.xs_l), lds_address(s.x[buf][pair] + (16 * k + 8 * half) * kRowX));
#pragma unroll
      for (int k = 0; k < 2; ++k)
        buffer_to_lds(bb, boff + (uint32_t)(64 * k * a.bs_l), lds_address(s.b[buf] + (32 * k + 4 * wave) * kRowB));
      if constexpr (OUT) {
        const u32x4 cb = rows_resource(cs, a.cs_l, left, 128);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          buffer_to_lds(cb, coff + (uint32_t)(64 * k * a.cs_l), lds_address(s.c[buf] + (32 * k + 4 * wave) * kRowB));
      }
      if (scalars) buffer_to_lds_u16(rows_resource(ds, a.ds_l, left, 1), doff, lds_address(s.dt[buf][pair]));
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = 32 * k + br, in = r < left ? 8 : 0;
        *(u32x4*)(s.b[buf] + (32 * k + 4 * wave) * kRowB + 8 * lane) = load8(bs + r * a.bs_l + 8 * bpart, in);
        if constexpr (OUT) *(u32x4*)(s.c[buf] + (32 * k + 4 * wave) * kRowB + 8 * lane) = load8(cs + r * a.cs_l + 8 * bpart, in);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *(u32x4*)(s.x[buf][pair] + (16 * k + 8 * half) * kRowX + 8 * lane) =
            load8(xs + (16 * k + xr) * a.xs_l + 8 * xpart, 16 * k + xr < left ? xcols : 0);
      if (scalars) s.dt[buf][pair][lane] = lane < left ? ds[lane * a.ds_l] : 0u;
    }
  };
  // the scalars of a chunk whose dt this wave has loaded
  auto prepare = [&](int64_t c0, int buf, int par) {   // lane = token
    ChunkScalars<OUT>& hs = s.h[par][pair];
    const bool in = c0 + lane < n;
    const float dt = in ? full_dt(h2f((uint16_t)s.dt[buf][pair][lane]) + bias) : 0.f;
    // (below 2^-4096 a decay leaves nothing of a carry; sums of more, or of minus
    // infinity, would leave differences without a value)
    double step = (double)av * (double)dt * 1.4426950408889634;
    step = in ? (step < -4096.0 ? -4096.0 : step) : 0.0;
    const double l = scan_add64(step);
    const double last = lane64(l, 63), tile = dpp_row_last64(l);
    const double e0 = lane64(l, 15), e1 = lane64(l, 31), e2 = lane64(l, 47);
    const double before = lane < 16 ? 0.0 : (lane < 32 ? e0 : (lane < 48 ? e1 : e2));
    const double up = last > 0.0 ? __builtin_floor(last < 1e6 ? last : 1e6) : 0.0;
    const float lh = (float)l, w = dt * __builtin_amdgcn_exp2f((float)(last - up - l));
    hs.w[lane] = w;
    if constexpr (OUT) {
      hs.lh[lane] = lh;
      hs.ll[lane] = __builtin_fabsf(lh) < __builtin_inff() ? (float)(l - (double)lh) : 0.f;
      hs.lt[lane] = (float)(l - before);
      hs.dt[lane] = dt;
      hs.ws[lane] = dt * __builtin_amdgcn_exp2f((float)(tile - l));
      hs.el[lane] = __builtin_amdgcn_exp2f(lh);
    }
    if constexpr (OUT) {
      const float dm = wave_max(finite_or_0(dt));
      if (lane == 0) hs.dtmax = dm;
    }
    if (lane == 0) {
      hs.tot = __builtin_amdgcn_exp2f((float)(last - up));
      hs.up = (float)up;
    }
    seg_log += last;
  };

  const int64_t chunks = (n + kChunk - 1) / kChunk;
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (k < chunks) load_chunk(k * kChunk, k);

  // the carry: S[16 nt + 4 lg + i][column] as st[nt][pt][i], 2^eS times its value.
  // Columns do not meet in any product, so each has powers of two of its own: a
  // large channel takes no bits from its neighbours.
  f32x4 st[8][2];
  int eS[2] = {0, 0};
  if constexpr (OUT) {
    // the row's only segment: the pool's own carry
    const float* base = seg == 0 && len <= t1 ? a.state + slot * a.H * a.P * 128 : sg.state + (seg * a.batch + b) * a.H * a.P * 128;
    const auto sb = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base + (h * a.P + pc) * 128), 0, (int)cols * 512, 0x00020000);
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)   // (zeros past the last column)
        st[nt][pt] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(sb, (pw + 16 * pt) * 512 + 16 * lg + 64 * nt, 0, 0));
  } else {
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) st[nt][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float sbound[2] = {0.f, 0.f};   // a bound of the carry's magnitudes, by column
  const int turned_at = bc_at(4 * lg + (lr >> 2), 4 * (lr & 3));   // for transposing reads of B
  float one = 1.0f;   // keeps the parts' differences mixed-precision fmas
  asm volatile("" : "+s"(one));
  uint32_t yoff[2];
#pragma unroll
  for (int pt = 0; pt < 2; ++pt) {
    const int p = 32 * half + 16 * pt + 4 * lg;
    yoff[pt] = p < cols ? (uint32_t)(2 * (lr * a.H * a.P + p)) : kOutside;
  }
  // a column's largest magnitude in units of st; an infinite coordinate must set
  // no scale
  auto largest = [&](float (&m)[2]) {
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      m[pt] = 0.f;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) m[pt] = __builtin_fmaxf(m[pt], __builtin_fabsf(st[nt][pt][i]));
      m[pt] = column_max(m[pt]);
    }
    if (__ballot(!(m[0] < __builtin_inff() && m[1] < __builtin_inff()))) {
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        m[pt] = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) m[pt] = __builtin_fmaxf(m[pt], __builtin_fabsf(finite_or_0(st[nt][pt][i])));
        m[pt] = column_max(m[pt]);
      }
    }
  };

  // One chunk token by token, in binary32 throughout: the carry in its own units
  // from here on.
  auto by_token = [&](int64_t c0, const ChunkScalars<OUT>& hs, const uint16_t* xt, const uint16_t* bt, const uint16_t* ct) {
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      const float undo = pow2(-eS[pt]);
      eS[pt] = 0;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) st[nt][pt] *= undo;
    }
    const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
    for (int t = 0; t < left; ++t) {
      const float dt = hs.dt[t];
      const float decay = __builtin_amdgcn_exp2f(t ? (hs.lh[t] - hs.lh[t - 1]) + (hs.ll[t] - hs.ll[t - 1]) : hs.lh[0]);
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        const float xv = h2f(xt[x_at(t, pw + 16 * pt)]), in = xv * dt;
        float acc = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float bv = h2f(bt[bc_at(t, 16 * nt + 4 * lg + i)]);
            st[nt][pt][i] = __builtin_fmaf(st[nt][pt][i], decay, in * bv);
            if constexpr (OUT) acc = __builtin_fmaf(st[nt][pt][i], h2f(ct[bc_at(t, 16 * nt + 4 * lg + i)]), acc);
          }
          __builtin_amdgcn_sched_barrier(0);   // few loads at a time: the registers are the chunks'
        }
        if constexpr (OUT) {
          acc = butterfly_add<5>(butterfly_add<4>(acc));
          if (lg == 0 && pw + 16 * pt < cols)
            a.y[((b * a.L + t0 + c0 + t) * a.H + h) * a.P + pc + pw + 16 * pt] = f2h(__builtin_fmaf(xv, dh, acc));
        }
      }
    }
    wait_vmcnt<0>();   // the next chunk, before these stores
  };

  // The first chunk has landed: behind its transfers are the carry's 16 loads,
  // which go on while the scalars are formed, or the transfers of the next.
  if constexpr (!ALIGNED) wait_vmcnt<0>();
  else if constexpr (OUT) wait_vmcnt<16>();
  else if (chunks < 2) wait_vmcnt<0>();
  else if (scalars) wait_vmcnt<7>();
  else wait_vmcnt<6>();
  bias = shift.value();
  dh = skip.value();
  if (scalars) prepare(0, 0, 0);
  __syncthreads();
  if constexpr (OUT) {   // here, so that the loop waits for no load of before it
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) asm volatile("" : "+v"(st[nt][pt]));
  }

  int buf = 0;
  for (int64_t ch = 0; ch < chunks; ++ch) {
    const int64_t c0 = ch * kChunk;
    const int par = (int)(ch & 1), next = buf + 1 < kBuffers ? buf + 1 : 0;
    const ChunkScalars<OUT>& hs = s.h[par][pair];
    const uint16_t *xt = s.x[buf][pair], *bt = s.b[buf], *ct = s.c[OUT ? buf : 0];
    const bool more = ch + kAhead < chunks;   // a chunk to be loaded: into the buffer that the last one left
    if (more) load_chunk(c0 + kAhead * kChunk, buf + kAhead < kBuffers ? buf + kAhead : buf + kAhead - kBuffers);

    // x fragments: tokens 16 T + 4 lg + r of column pw + 16 pt
    f16x4 xf[2][4];
    uint32_t xm = 0;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int T = 0; T < 4; ++T) {
        xf[pt][T] = read_transposed(xt + 16 * T * kRowX + x_at(4 * lg + (lr >> 2), 32 * half + 16 * pt + 4 * (lr & 3)));
        xm = max_magnitudes(xm, __builtin_bit_cast(u32x2, xf[pt][T]));
      }

    // 8 coordinates of row 16 tile + lr of B or C in the order of the carry's
    // fragments: 32 kk + 4 lg + ..., and 16 further
    const int row_at = bc_at(lr, 4 * lg);
    auto row_fragment = [&](const uint16_t* m, int tile, int kk) {
      const uint16_t* r = m + 16 * tile * kRowB;
      return join(*(const f16x4*)(r + (row_at ^ (32 * kk))), *(const f16x4*)(r + (row_at ^ (32 * kk + 16))));
    };
    // The same in reads of their own (volatile): paired by the compiler, the
    // reads of two tiles meet on the same banks (1,000 of a chunk's LDS cycles).
    auto row_fragment_alone = [&](const uint16_t* m, int tile, int kk) {
      const uint16_t* r = m + 16 * tile * kRowB;
      return join(*(const volatile lds_f16x4*)(r + (row_at ^ (32 * kk))),
                  *(const volatile lds_f16x4*)(r + (row_at ^ (32 * kk + 16))));
    };
    // A non-finite x must not reach earlier tokens, which the matrix products would
    // let it do (0 * inf); and where the carry grows (a positive A) the last tokens'
    // weights would set the first ones' scale: such a chunk token by token.
    bool odd = OUT && (__ballot(non_finite_half(xm)) != 0 || hs.tot > 1.0f || hs.up > 0.f);
    if constexpr (OUT) {
      // ---- C B^T, the same for all heads: two waves without scalars two tiles, the others one.
      // Tile (j, i): rows tokens 16 j + 4 lg + r (B), columns tokens 16 i + lr (C).
      float gm = 0.f;
      auto score_tile = [&](int at) {
        const int i = at < 1 ? 0 : (at < 3 ? 1 : (at < 6 ? 2 : 3)), j = at - i * (i + 1) / 2;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) acc = mfma(row_fragment(bt, j, kk), row_fragment(ct, i, kk), acc);
        s.scores[at][lane] = acc;
#pragma unroll
        for (int k = 0; k < 4; ++k) gm = __builtin_fmaxf(gm, __builtin_fabsf(finite_or_0(acc[k])));
      };
      score_tile(wave);
      if (wave == 1 || wave == 3) score_tile(wave == 1 ? 8 : 9);
      gm = wave_max(gm);
      if (lane == 0) s.gmax[wave] = gm;

      f32x4 acc[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) acc[i][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
      float smax[2];
      largest(smax);
      int kS[2];   // in units of st
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        sbound[pt] = __builtin_ldexpf(smax[pt], -eS[pt]);
        kS[pt] = 13 - exponent_of(smax[pt]) > 100 ? 100 : 13 - exponent_of(smax[pt]);
      }
      // (so would one of carries whose products leave binary32)
      odd = odd || __ballot(sbound[0] > 0x1p40f || sbound[1] > 0x1p40f) != 0;
      if (!odd) {
        // ---- S C_t: rows = columns of x, columns = tokens
        float ss[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          ss[pt] = pow2(kS[pt]);
          s.undo[wave][16 * pt + lr] = __builtin_ldexpf(1.0f, -kS[pt] - eS[pt]);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          Split f[2];
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = st[2 * kk + (i >> 2)][pt][i & 3];
            f[pt] = split8(v, ss[pt]);
          }
          f16x8 cf[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) cf[i] = row_fragment_alone(ct, i, kk);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(f[pt].hi, cf[i], acc[i][pt]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(f[pt].lo, cf[i], acc[i][pt]);
        }
        // (written and read by this wave alone)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          const f32x4 u = *(const f32x4*)(s.undo[wave] + 16 * pt + 4 * lg);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][pt][r] *= u[r];
        }
      } else {
        by_token(c0, hs, xt, bt, ct);
      }
      __syncthreads();   // the scores are there

      if (!odd) {
        // ---- masked scores and their product with x.  Below the diagonal
        // tiles the decay is 2^(l_t - r_j) 2^(r_j - l_s), no factor above 1;
        // D joins the diagonal.
        float gmax = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) gmax = __builtin_fmaxf(gmax, s.gmax[k]);
        const float mb = gmax * hs.dtmax + __builtin_fabsf(dh);   // bounds the finite weights
        // Those below 2^14, so that a non-finite score or step, which is in some
        // tokens' weights only, leaves the others' bits (an infinite D is in all).
        // (No power above 24: what that leaves out is nothing in a readout.)
        int km = mb < __builtin_inff() ? 13 - exponent_of(mb) : 0;
        km = km > 24 ? 24 : km;
        km = __builtin_amdgcn_readfirstlane(km);
        const float scale = pow2(km), back = pow2(-km), fkm = (float)km;
        float dk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) dk[k] = 4 * lg + k == lr ? dh * scale : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float th = hs.lh[16 * i + lr], tl = hs.ll[16 * i + lr] + fkm;
          float v[16];
#pragma unroll
          for (int j = 0; j < i; ++j) {
            const float ft = __builtin_amdgcn_exp2f((th - hs.lh[16 * j + 15]) + (tl - hs.ll[16 * j + 15]));
            const f32x4 gt = s.scores[i * (i + 1) / 2 + j][lane], ws = *(const f32x4*)(hs.ws + 16 * j + 4 * lg);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[4 * j + k] = (gt[k] * ws[k]) * ft;
          }
          {
            const f32x4 gt = s.scores[i * (i + 1) / 2 + i][lane];
            const f32x4 sd = *(const f32x4*)(hs.dt + 16 * i + 4 * lg), sl = *(const f32x4*)(hs.lt + 16 * i + 4 * lg);
            const float tt = hs.lt[16 * i + lr] + fkm;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float e = __builtin_amdgcn_exp2f(tt - sl[k]);
              float m = __builtin_fmaf(gt[k] * sd[k], e, dk[k]);
              asm volatile("" : "+v"(m));   // formed by all lanes, without a branch around it
              v[4 * i + k] = 4 * lg + k <= lr ? m : 0.f;
            }
          }
#pragma unroll
          for (int k = 4 * i + 4; k < 16; ++k) v[k] = 0.f;
          const float f = hs.el[16 * i + lr] * (scale * (1 << kLeast));
          Split3 m[2];
#pragma unroll
          for (int kk = 0; kk <= i / 2; ++kk) m[kk] = split8_3(v + 8 * kk, one);
          auto add = [&](f16x8 Split3::*part) {
#pragma unroll
            for (int kk = 0; kk <= i / 2; ++kk)
#pragma unroll
              for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(join(xf[pt][2 * kk], xf[pt][2 * kk + 1]), m[kk].*part, acc[i][pt]);
          };
          auto rescale = [&](float by) {
#pragma unroll
            for (int pt = 0; pt < 2; ++pt)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][pt][r] *= by;
          };
          rescale(f);
          add(&Split3::least);
          rescale(1.0f / (1 << kLeast));
          add(&Split3::lo);
          add(&Split3::hi);
        }
        const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
        uint16_t* yc = a.y + ((b * a.L + t0 + c0) * a.H + h) * a.P + pc;
        const auto yb = rows_buffer(yc, a.H * a.P, left, (int)cols);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            f16x4 out;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float q = acc[i][pt][r] * back;
              asm volatile("" : "+v"(q));   // rounded to binary32 first in every instance
              out[r] = (_Float16)q;
            }
            if constexpr (ALIGNED) {
              __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, out), yb, yoff[pt] + (uint32_t)(32 * i * a.H * a.P), 0, 0);
            } else {
              const int p = 32 * half + 16 * pt + 4 * lg;
              const s16x4v bits = __builtin_bit_cast(s16x4v, out);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (16 * i + lr < left && p + r < cols) yc[(16 * i + lr) * a.H * a.P + p + r] = (uint16_t)bits[r];
            }
          }
        }
      }
    }

    // ---- the carry after the chunk: a column's x w 2^e1 below 2^14, unless a
    // bound of its carry (the decayed one and 64 products) would leave binary32.
    if (!odd) {
      const float tot = hs.tot;
      const int up = OUT ? 0 : (int)hs.up;   // (a growing chunk is an odd one with readouts)
      float xw[2][16], mx[2], keep[2], sx[2];
      int d[2];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        mx[pt] = 0.f;
#pragma unroll
        for (int T = 0; T < 4; ++T) {
          const f32x4 w = *(const f32x4*)(hs.w + 16 * T + 4 * lg);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            xw[pt][4 * T + i] = __builtin_fmaf((float)xf[pt][T][i], w[i], 0.f);   // (one mixed fma)
            mx[pt] = __builtin_fmaxf(mx[pt], __builtin_fabsf(xw[pt][4 * T + i]));
          }
        }
        mx[pt] = column_max(mx[pt]);
        sbound[pt] = __builtin_ldexpf(__builtin_fmaf(sbound[pt], tot, 64.0f * 65504.0f * mx[pt]), up);
        const int most = 120 - (sbound[pt] < 0x1p120f ? exponent_of(sbound[pt]) : 121);
        int e1 = 13 - exponent_of(mx[pt]);
        e1 = e1 < most ? e1 : most;
        e1 = mx[pt] > 0.f && mx[pt] < __builtin_inff() ? e1 : eS[pt];
        e1 = e1 < 110 ? (e1 > -110 ? e1 : -110) : 110;
        d[pt] = e1 - eS[pt];
        eS[pt] = e1 - up;
        keep[pt] = __builtin_ldexpf(tot, d[pt]);
        sx[pt] = pow2(e1);
      }
      // (a factor past binary32 would make a carry of zero a NaN)
      if (__ballot(d[0] > 100 || d[1] > 100 || d[0] < -100 || d[1] < -100)) {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[nt][pt][i] = __builtin_ldexpf(st[nt][pt][i] * tot, d[pt]);
        keep[0] = keep[1] = 1.0f;
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[nt][pt][i] *= keep[pt];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        Split f[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) f[pt] = split8(xw[pt] + 8 * kk, sx[pt]);
        const uint16_t* r = bt + 32 * kk * kRowB;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const f16x8 bf = join(read_transposed(r + (turned_at ^ (16 * nt))), read_transposed(r + 16 * kRowB + (turned_at ^ (16 * nt))));
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) st[nt][pt] = mfma(bf, f[pt].hi, st[nt][pt]);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) st[nt][pt] = mfma(bf, f[pt].lo, st[nt][pt]);
        }
      }
      // The next chunk has landed: behind its transfers are the 8 stores of
      // readouts, or the transfers of the chunk after it.
      if constexpr (ALIGNED) {
        if constexpr (OUT) {
          wait_vmcnt<8>();
        } else {
          if (!more) wait_vmcnt<0>();
          else if (scalars) wait_vmcnt<7>();
          else wait_vmcnt<6>();
        }
      }
    }
    if (scalars && ch + 1 < chunks) prepare(c0 + kChunk, next, par ^ 1);
    __syncthreads();
    buf = next;
  }

  if (!OUT || len <= t1) {
    const int64_t base = OUT ? slot * a.H + h : ((seg + 1) * a.batch + b) * a.H + h;
    float* dst = OUT ? a.state : sg.state;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
      if (pw + 16 * pt < cols) {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[nt][pt][i] = __builtin_ldexpf(st[nt][pt][i], -eS[pt]);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
          *(f32x4*)(dst + (base * a.P + pc + pw + 16 * pt) * 128 + 16 * nt + 4 * lg) = st[nt][pt];
      }
    if (!OUT && live && scalars && pc == 0 && lane == 0) {
      const double e = __builtin_fmin(__builtin_fmax(__builtin_floor(seg_log), -1000.0), 1000.0);
      sg.decay[base] = f32x2{__builtin_amdgcn_exp2f((float)(seg_log - e)), (float)e};
    }
  }
}

// The carries before each segment, of rows of more than one: a running fma over
// the segments' additions, four values a thread, eight loads in flight.  Bound
// by memory: 8 segments of 128 heads of 64 (67 MB) 12.7 us, 5.3 TB/s.
__global__ __launch_bounds__(256) void k_full_join(FullArgs a, Segments sg) {
  const int64_t b = blockIdx.y, i = (int64_t)blockIdx.x * 256 + threadIdx.x, per_row = a.H * a.P * 32;
  if (i >= per_row) return;
  const FullRow fr = full_row(a, b);
  const int64_t slot = fr.slot, len = fr.len;
  const int64_t started = (len + sg.tokens - 1) / sg.tokens;
  if (started < 2) return;
  const int64_t h = i / (a.P * 32);
  f32x4 cur = *(const f32x4*)(a.state + (slot * per_row + i) * 4);
  f32x4* at = (f32x4*)sg.state + b * per_row + i;
  const int64_t step = a.batch * per_row;
  at[0] = cur;
  for (int64_t q0 = 1; q0 < started; q0 += 8) {
    f32x4 v[8];
    f32x2 d[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (q0 + k < started) {
        v[k] = at[(q0 + k) * step];
        d[k] = sg.decay[((q0 + k) * a.batch + b) * a.H + h];
      }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (q0 + k < started) {
#pragma unroll
        for (int e = 0; e < 4; ++e) cur[e] = __builtin_fmaf(__builtin_ldexpf(cur[e], (int)d[k][1]), d[k][0], v[k][e]);
        at[(q0 + k) * step] = cur;
      }
  }
}

}  // namespace m2r

using namespace m2r;

namespace m2r {

// How many segments a call's tokens are split into: a workgroup on each of 256
// compute units at most.
Segments full_segments(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G) {
  const int64_t hpg = H / G, blocks = (hpg * ((P + 63) / 64) + 3) / 4, chunks = (L + kChunk - 1) / kChunk;
  const int64_t groups = blocks * G * batch;
  int64_t want = groups < 256 ? 256 / groups : 1;
  want = want < chunks ? want : chunks;
  const int64_t per = (chunks + want - 1) / want;
  return Segments{per * kChunk, (int)((chunks + per - 1) / per), nullptr, nullptr, false};
}

int64_t full_chunks_workspace(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G) {
  const Segments sg = full_segments(batch, L, H, P, G);
  return sg.count > 1 ? (int64_t)sg.count * batch * H * (P * 128 + 2) * 4 : 0;
}

hipError_t launch_full_chunks(const FullArgs& a, void* workspace, hipStream_t stream) {
  Segments sg = full_segments(a.batch, a.L, a.H, a.P, a.G);
  const int64_t hpg = a.H / a.G, blocks = (hpg * ((a.P + 63) / 64) + 3) / 4;
  if (sg.count > 1) {
    sg.state = (float*)workspace;
    sg.decay = (f32x2*)(sg.state + (int64_t)sg.count * a.batch * a.H * a.P * 128);
  }
  // 16-byte pieces through buffers: rows that do not overlap, and 64 of them
  // within 31-bit offsets
  const int64_t far = (int64_t)1 << 23, dense = a.H * a.P;
  const bool aligned = a.P % 8 == 0 && ((a.xs_b | a.xs_l | a.bs_b | a.bs_l | a.cs_b | a.cs_l) & 7) == 0 &&
                       (((uintptr_t)a.x | (uintptr_t)a.Bm | (uintptr_t)a.Cm | (uintptr_t)a.y) & 15) == 0 &&
                       a.xs_l >= dense && a.bs_l >= a.G * 128 && a.cs_l >= a.G * 128 && a.ds_l >= a.H &&
                       a.xs_l < far && a.bs_l < far && a.cs_l < far && a.ds_l < far;
  // Somewhat more workgroups than compute units: the rows that take longest
  // start first.  us for ragged rows of 32 workgroups each, so / as they come:
  // 9 of up to 901 tokens 128 / 154, 12 of up to 901 141 / 166, 20 of up to 600
  // 173 / 182; more rows even out by themselves, and their short ones, which
  // mostly move carries, run better among long ones: 40 of up to 300 218 / 209,
  // 64 of up to 150 253 / 221.
  const int64_t groups = blocks * a.G * a.batch;
  sg.longest_first = a.lengths && a.batch <= 64 && groups > 256 && groups <= 768;
  const dim3 block(512);
  dim3 grid((unsigned)(blocks * a.G), (unsigned)a.batch, (unsigned)sg.count);
  if (sg.count > 1) {
    grid.z = sg.count - 1;
    if (aligned) hipLaunchKernelGGL((k_full_chunks<true, false>), grid, block, 0, stream, a, sg);
    else hipLaunchKernelGGL((k_full_chunks<false, false>), grid, block, 0, stream, a, sg);
    const dim3 join((unsigned)((a.H * a.P * 32 + 255) / 256), (unsigned)a.batch);
    hipLaunchKernelGGL(k_full_join, join, dim3(256), 0, stream, a, sg);
    grid.z = sg.count;
  }
  if (aligned) hipLaunchKernelGGL((k_full_chunks<true, true>), grid, block, 0, stream, a, sg);
  else hipLaunchKernelGGL((k_full_chunks<false, true>), grid, block, 0, stream, a, sg);
  return hipGetLastError();
}

}  // namespace m2r
