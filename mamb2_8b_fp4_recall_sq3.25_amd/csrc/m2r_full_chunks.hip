// Scan with a full-precision carry over many tokens, on the matrix cores: the
// recurrence of m2r_full.hip in chunks of 64 tokens.  With l_t the running sum
// of A dt inside a chunk, S the carry before it and S' the carry after it,
//   y_t = sum_{s <= t} (C_t . B_s) exp(l_t - l_s) dt_s x_s + exp(l_t) S C_t + D x_t
//   S'  = exp(l_63) S + sum_s exp(l_63 - l_s) dt_s x_s (x) B_s.
#include "m2r_full.h"
#include "m2r_abi_util.h"

namespace m2r {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4v lds_s16x4;

constexpr int kChunk = 64;
// LDS row pitches in binary16 elements.  C is read as 16 bytes of 16 rows (a
// pitch of 4 banks past a multiple of 64 puts them on all banks once), B
// by transposing reads of 4 rows by 32 bytes per 16 lanes (8 banks apart).
// x comes by direct transfers (64 lanes x 16 bytes in a row), so its rows are
// dense and their 16-byte pieces are exchanged instead: the piece of columns
// 8 c .. 8 c + 7 of row r stands at c ^ x_turn(r), which spreads the 4 rows x
// 32 bytes that 16 lanes read over all banks.
constexpr int kPitchC = 136, kPitchB = 144, kPitchX = 64;
__device__ __forceinline__ int x_turn(int row) { return ((row >> 1) & 3) << 1; }
__device__ __forceinline__ int x_at(int row, int col) { return row * kPitchX + 8 * ((col >> 3) ^ x_turn(row)) + (col & 7); }

// What the heads' tokens need besides B, C and x.  l is the running sum of
// A dt log2(e) over the chunk, r_j its value at the last token of the 16-token
// tile j; powers are of two.
struct ChunkScalars {
  float lh[kChunk], ll[kChunk];   // l as a sum of two binary32
  float lt[kChunk];               // l - r of the tile before
  float dt[kChunk];
  float ws[kChunk];               // dt 2^(r_tile - l)
  float w[kChunk];                // dt 2^(l_63 - l)
  float el[kChunk];               // 2^l
  float tot, wmax, dtmax, unused; // 2^l_63, the largest w and dt
};

struct ChunkShared {
  uint16_t c[kChunk * kPitchC];          // each 32 coordinates in the order of the carry's fragments
  uint16_t b[2][kChunk * kPitchB];
  uint16_t x[2][4][kChunk * kPitchX];
  f32x4 scores[10][64];                  // (C B^T) tiles on and below the diagonal, by lane
  ChunkScalars h[2][4];
  float gmax[8];                         // largest score, by wave
  uint32_t bmax[2][8];                   // largest magnitude of B as binary16, by wave
};

struct Segments {
  int64_t tokens;     // of a segment, a multiple of kChunk
  int count;
  // For rows that go on past their first segment, [count, batch, H, P, 128]:
  // 0 the row's first carry (the pool's own is overwritten by the last segment
  // while others still start), q > 0 first what segment q - 1 adds to a zero
  // carry, then (k_full_join) the carry before segment q; and the decay over
  // segment q - 1.
  float* state;
  float* decay;       // [count, batch, H]
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
// floor(log2 v) of a positive normal v (-127 for zero and subnormals).
__device__ __forceinline__ int exponent_of(float v) { return ((__builtin_bit_cast(int, v) >> 23) & 255) - 127; }
__device__ __forceinline__ float pow2(int k) { return __builtin_ldexpf(1.0f, k); }

// v as the sum of two binary16, in units in which the largest value has the
// exponent 14: the first carries 11 bits, the second the next 11 (whatever is
// left above 2^-25), so that a product of a binary16 factor with both keeps
// 22 bits, and is summed in binary32 by the matrix instruction.  `scale`, a
// power of two, comes with the conversions: v scale - high is one mixed fma.
struct Split { f16x8 hi, lo; };
__device__ __forceinline__ Split split8(const float* v, float one) {   // one: 1, not known to the compiler
  Split s;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 h = __builtin_convertvector((f32x2{v[j], v[j + 1]}), f16x2);
    const f16x2 l = __builtin_convertvector(
        (f32x2{__builtin_fmaf(v[j], one, -(float)h[0]), __builtin_fmaf(v[j + 1], one, -(float)h[1])}), f16x2);
    s.hi[j] = h[0];
    s.hi[j + 1] = h[1];
    s.lo[j] = l[0];
    s.lo[j + 1] = l[1];
  }
  return s;
}
__device__ __forceinline__ Split split8_scaled(const float* v, float scale) {
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

// Direct transfer of 16 bytes a lane to lds + 16 lane, from `off` into the
// buffer; zeros for offsets outside.  The caller waits (wait_vmcnt).
__device__ __forceinline__ void buffer_to_lds(u32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc),
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
__device__ __forceinline__ uint32_t wave_max_half(uint32_t m) {
  const uint32_t lo = m & 0xffffu, hi = m >> 16;
  return wave_max_bits(lo > hi ? lo : hi);
}
// A workgroup steps four blocks of 64 columns (a head's channels) of one
// group, two waves each, over one segment of one batch row's tokens.  OUT:
// readouts and the pool's carry; else what the segment adds to a zero carry.
template <bool ALIGNED, bool OUT>
__global__ __launch_bounds__(512, 2) void k_full_chunks(FullArgs a, Segments sg) {
  __shared__ ChunkShared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), pair = wave >> 1, half = wave & 1;
  const int lr = lane & 15, lg = lane >> 4;
  const int hpg = (int)(a.H / a.G), per_head = (int)((a.P + 63) / 64), blocks = (hpg * per_head + 3) / 4;
  const int g = blockIdx.x / blocks, blk = blockIdx.x - g * blocks;
  const int64_t b = blockIdx.y, seg = blockIdx.z;

  const int64_t slot = full_slot(a, b);
  const int64_t len = slot < 0 ? 0 : full_length(a, b);
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

  const float av = a.A[h], dh = load_param(a.D, a.d_f32, (int)h), bias = load_param(a.dt_bias, a.db_f32, (int)h);
  double seg_log = 0.0;   // the segment's decay so far, as a power of two

  // the loads of a chunk: B and C two, x four 16-byte pieces a thread
  u32x4 rb[2], rc[2], rx[ALIGNED ? 1 : 4];
  uint16_t rdt = 0;
  // x: transfer k of a wave fills rows 16 k + 8 half ... + 7, the lane's piece
  // of them at its turned place
  const int br = tid >> 4, bpart = tid & 15, xr = 8 * half + (lane >> 3), xpart = (lane & 7) ^ x_turn(lane >> 3);
  const uint16_t *bp = a.Bm + b * a.bs_b + t0 * a.bs_l + g * 128, *cp = a.Cm + b * a.cs_b + t0 * a.cs_l + g * 128;
  const uint16_t *xp = a.x + b * a.xs_b + t0 * a.xs_l + h * a.P + pc, *dp = a.dt + b * a.ds_b + t0 * a.ds_l + h;
  const int xcols = (int)cols - 8 * xpart;
  const uint32_t xoff = xcols > 0 ? (uint32_t)(2 * (xr * a.xs_l + 8 * xpart)) : kOutside;
  const uint32_t boff = (uint32_t)(2 * (br * a.bs_l + 8 * bpart)), coff = (uint32_t)(2 * (br * a.cs_l + 8 * bpart));
  // the wave that prepares its pair's scalars: one of the two on each SIMD
  const bool scalars = half == pair >> 1;
  auto load_chunk = [&](int64_t c0, int par) {   // tokens t0 + c0 ...: the pointers stand there
    const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
    if constexpr (ALIGNED) {
      const auto bb = rows_buffer(bp, a.bs_l, left, 128), cb = rows_buffer(cp, a.cs_l, left, 128);
      const auto db = rows_buffer(dp, a.ds_l, left, 1);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        rb[k] = __builtin_amdgcn_raw_buffer_load_b128(bb, boff + (uint32_t)(64 * k * a.bs_l), 0, 0);
        if (OUT) rc[k] = __builtin_amdgcn_raw_buffer_load_b128(cb, coff + (uint32_t)(64 * k * a.cs_l), 0, 0);
      }
      if (scalars) rdt = __builtin_amdgcn_raw_buffer_load_b16(db, (uint32_t)(2 * lane * a.ds_l), 0, 0);
      const u32x4 xb = rows_resource(xp, a.xs_l, left, (int)cols);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        buffer_to_lds(xb, xoff + (uint32_t)(32 * k * a.xs_l), lds_address(s.x[par][pair] + (16 * k + 8 * half) * kPitchX));
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = 32 * k + br, in = r < left ? 8 : 0;
        rb[k] = load8(bp + r * a.bs_l + 8 * bpart, in);
        if (OUT) rc[k] = load8(cp + r * a.cs_l + 8 * bpart, in);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        rx[k] = load8(xp + (16 * k + xr) * a.xs_l + 8 * xpart, 16 * k + xr < left ? xcols : 0);
      if (scalars) rdt = lane < left ? dp[lane * a.ds_l] : 0;
    }
    bp += kChunk * a.bs_l;
    cp += kChunk * a.cs_l;
    xp += kChunk * a.xs_l;
    dp += kChunk * a.ds_l;
  };
  // the loaded chunk into LDS (B, x and the scalars: buffer `par`)
  auto store_chunk = [&](int64_t c0, int par) {
    uint32_t bm = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = 32 * k + br;
      *(u32x4*)(s.b[par] + r * kPitchB + 8 * bpart) = rb[k];
      bm = max_magnitudes(bm, rb[k]);
      if (OUT) {
        // coordinates 32 kk + 16 T + 4 q + i of a row stand at 32 kk + 8 q + 4 T + i
        const int kk = bpart >> 2, T = (bpart >> 1) & 1, q = 2 * (bpart & 1);
        uint16_t* d = s.c + r * kPitchC + 32 * kk + 8 * q + 4 * T;
        *(u32x2*)d = u32x2{rc[k][0], rc[k][1]};
        *(u32x2*)(d + 8) = u32x2{rc[k][2], rc[k][3]};
      }
    }
    if constexpr (ALIGNED) {
      wait_vmcnt<0>();   // the transfers have landed
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) *(u32x4*)(s.x[par][pair] + (16 * k + 8 * half) * kPitchX + 8 * lane) = rx[k];
    }
    bm = wave_max_half(bm);
    if (lane == 0) s.bmax[par][wave] = bm;
    if (scalars) {   // lane = token
      ChunkScalars& hs = s.h[par][pair];
      const float dt = c0 + lane < n ? full_dt(h2f(rdt) + bias) : 0.f;
      const double l = scan_add64((double)av * (double)dt * 1.4426950408889634);
      const double last = lane64(l, 63), tile = dpp_row_last64(l);
      const double e0 = lane64(l, 15), e1 = lane64(l, 31), e2 = lane64(l, 47);
      const double before = lane < 16 ? 0.0 : (lane < 32 ? e0 : (lane < 48 ? e1 : e2));
      const float lh = (float)l, w = dt * __builtin_amdgcn_exp2f((float)(last - l));
      hs.lh[lane] = lh;
      hs.ll[lane] = __builtin_fabsf(lh) < __builtin_inff() ? (float)(l - (double)lh) : 0.f;
      hs.lt[lane] = (float)(l - before);
      hs.dt[lane] = dt;
      hs.ws[lane] = dt * __builtin_amdgcn_exp2f((float)(tile - l));
      hs.w[lane] = w;
      hs.el[lane] = __builtin_amdgcn_exp2f(lh);
      const float wm = wave_max(w), dm = wave_max(dt);
      if (lane == 0) {
        hs.tot = __builtin_amdgcn_exp2f((float)last);
        hs.wmax = wm;
        hs.dtmax = dm;
      }
      seg_log += last;
    }
  };

  load_chunk(0, 0);

  // the carry: S[16 nt + 4 lg + i][column] as st[nt][pt][i], 2^-eS times its value
  f32x4 st[8][2];
  int eS = 0;
  {
    // the row's only segment: the pool's own carry
    const float* base = seg == 0 && len <= t1 ? a.state + slot * a.H * a.P * 128 : sg.state + (seg * a.batch + b) * a.H * a.P * 128;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      const float* src = base + (h * a.P + pc + pw + 16 * pt) * 128 + 4 * lg;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
        st[nt][pt] = OUT && pw + 16 * pt < cols ? *(const f32x4*)(src + 16 * nt) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  float one = 1.0f;   // keeps the halves' differences mixed-precision fmas
  asm volatile("" : "+s"(one));
  uint32_t yoff[2];
#pragma unroll
  for (int pt = 0; pt < 2; ++pt) {
    const int p = 32 * half + 16 * pt + 4 * lg;
    yoff[pt] = p < cols ? (uint32_t)(2 * (lr * a.H * a.P + p)) : kOutside;
  }
  // a bound of the carry's magnitudes, 2^eb
  float smax = 0.f;
#pragma unroll
  for (int nt = 0; nt < 8; ++nt)
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = __builtin_fabsf(st[nt][pt][i]);
        smax = __builtin_fmaxf(smax, v < __builtin_inff() ? v : 0.f);   // an infinite channel sets no scale
      }
  smax = wave_max(smax);
  int eb = exponent_of(smax) + 1;

  store_chunk(0, 0);
  __syncthreads();

  const int64_t chunks = (n + kChunk - 1) / kChunk;
  for (int64_t ch = 0; ch < chunks; ++ch) {
    const int64_t c0 = ch * kChunk;
    const int par = (int)(ch & 1);
    const ChunkScalars& hs = s.h[par][pair];
    const uint16_t *xt = s.x[par][pair], *bt = s.b[par];
    if (ch + 1 < chunks) load_chunk(c0 + kChunk, par ^ 1);

    // x fragments: tokens 16 T + 4 lg + r of column pw + 16 pt
    f16x4 xf[2][4];
    uint32_t xm = 0;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int T = 0; T < 4; ++T) {
        xf[pt][T] = read_transposed(xt + 16 * T * kPitchX + x_at(4 * lg + (lr >> 2), 32 * half + 16 * pt + 4 * (lr & 3)));
        xm = max_magnitudes(xm, __builtin_bit_cast(u32x2, xf[pt][T]));
      }
    xm = wave_max_half(xm);

    const bool odd = OUT && xm >= 0x7c00u;
    if constexpr (OUT) {
      // ---- C B^T, the same for all heads: two waves without scalars two tiles, the others one.
      // Tile (j, i): rows tokens 16 j + 4 lg + r (B), columns tokens 16 i + lr (C).
      float gm = 0.f;
      auto score_tile = [&](int at) {
        const int i = at < 1 ? 0 : (at < 3 ? 1 : (at < 6 ? 2 : 3)), j = at - i * (i + 1) / 2;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        const uint16_t *cr = s.c + (16 * i + lr) * kPitchC + 8 * lg, *r = bt + (16 * j + lr) * kPitchB + 4 * lg;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          acc = mfma(join(*(const f16x4*)(r + 32 * kk), *(const f16x4*)(r + 32 * kk + 16)), *(const f16x8*)(cr + 32 * kk), acc);
        s.scores[at][lane] = acc;
#pragma unroll
        for (int k = 0; k < 4; ++k) gm = __builtin_fmaxf(gm, __builtin_fabsf(acc[k]));
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
      const int kS = 14 - eb > 100 ? 100 : 14 - eb;
      if (odd) {
        // A non-finite x must not reach earlier tokens, which the matrix
        // products would let it do (0 * inf): this chunk token by token.
        const float undo = pow2(-eS);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) st[nt][pt] *= undo;
        const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
        for (int t = 0; t < left; ++t) {
          const float dt = hs.dt[t];
          const float decay = __builtin_amdgcn_exp2f(t ? (hs.lh[t] - hs.lh[t - 1]) + (hs.ll[t] - hs.ll[t - 1]) : hs.lh[0]);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            const float xv = h2f(xt[x_at(t, pw + 16 * pt)]), in = xv * dt;
            float acc = 0.f;
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float bv = h2f(bt[t * kPitchB + 16 * nt + 4 * lg + i]);
                const float cv = h2f(s.c[t * kPitchC + 32 * (nt >> 1) + 8 * lg + 4 * (nt & 1) + i]);
                st[nt][pt][i] = __builtin_fmaf(st[nt][pt][i], decay, in * bv);
                acc = __builtin_fmaf(st[nt][pt][i], cv, acc);
              }
            acc = butterfly_add<5>(butterfly_add<4>(acc));
            if (lg == 0 && pw + 16 * pt < cols)
              a.y[((b * a.L + t0 + c0 + t) * a.H + h) * a.P + pc + pw + 16 * pt] = f2h(__builtin_fmaf(xv, dh, acc));
          }
        }
        smax = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = __builtin_fabsf(st[nt][pt][i]);
              smax = __builtin_fmaxf(smax, v < __builtin_inff() ? v : 0.f);
            }
        smax = wave_max(smax);
        eb = exponent_of(smax) + 1;
        eS = 0;
      } else {
        // ---- S C_t: rows = columns of x, columns = tokens
        const float ss = pow2(kS - eS);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          Split f[2];
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = st[2 * kk + (i >> 2)][pt][i & 3];
            f[pt] = split8_scaled(v, ss);
          }
          f16x8 cf[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) cf[i] = *(const f16x8*)(s.c + (16 * i + lr) * kPitchC + 32 * kk + 8 * lg);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(f[pt].hi, cf[i], acc[i][pt]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(f[pt].lo, cf[i], acc[i][pt]);
        }
      }
      __syncthreads();   // the scores are there

      if (!odd) {
        // ---- masked scores and their product with x.  Below the diagonal
        // tiles the decay is 2^(l_t - r_j) 2^(r_j - l_s), no factor above 1
        // for a negative A; D joins the diagonal.
        float gmax = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) gmax = __builtin_fmaxf(gmax, s.gmax[k]);
        const float tot = hs.tot;
        float mb = gmax * hs.dtmax * (tot > 1.f ? tot : 1.f) + __builtin_fabsf(dh);   // bounds the weights
        // Weights below 2^15.  Below 2^-25 one times any x is nothing in the
        // readout; and without a finite bound there is no scale to choose.
        int km = mb < __builtin_inff() ? 13 - exponent_of(mb) : 0;
        km = km > 40 ? 40 : km;
        km = __builtin_amdgcn_readfirstlane(km);
        const float scale = pow2(km), back = pow2(-km), fkm = (float)km;
        float dk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) dk[k] = 4 * lg + k == lr ? dh * scale : 0.f;
        const int left = (int)(n - c0 < kChunk ? n - c0 : kChunk);
        uint16_t* yc = a.y + ((b * a.L + t0 + c0) * a.H + h) * a.P + pc;
        const auto yb = rows_buffer(yc, a.H * a.P, left, (int)cols);
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
          const float f = __builtin_ldexpf(hs.el[16 * i + lr], km - kS);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][pt][r] *= f;
#pragma unroll
          for (int kk = 0; kk <= i / 2; ++kk) {
            const Split m = split8(v + 8 * kk, one);
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(join(xf[pt][2 * kk], xf[pt][2 * kk + 1]), m.hi, acc[i][pt]);
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) acc[i][pt] = mfma(join(xf[pt][2 * kk], xf[pt][2 * kk + 1]), m.lo, acc[i][pt]);
          }
        }
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

    // ---- the carry after the chunk.  The bound: the decayed carry's and 64
    // products', each factor below twice its power of two.
    if (!odd) {
      uint32_t bm8 = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) bm8 = bm8 > s.bmax[par][k] ? bm8 : s.bmax[par][k];
      const float tot = hs.tot, wmax = hs.wmax;
      const int ex = xm >= 0x7c00u ? 16 : exponent_of(h2f((uint16_t)xm)), ebm = bm8 >= 0x7c00u ? 16 : exponent_of(h2f((uint16_t)bm8));
      const int old = eb + (tot < __builtin_inff() ? exponent_of(tot) + 1 : 128);
      int add = ex + exponent_of(wmax) + ebm + 9;
      if (!(wmax < __builtin_inff())) add = 128;
      eb = (old > add ? old : add) + 1;
      eb = eb > 128 ? 128 : (eb < -126 ? -126 : eb);
      // x w 2^e1 below 2^15, unless the carry would leave binary32
      int e1 = eS;
      if (xm && wmax > 0.f && wmax < __builtin_inff()) {
        e1 = 13 - ex - exponent_of(wmax);
        e1 = e1 < 110 - eb ? e1 : 110 - eb;
        e1 = e1 < 110 ? (e1 > -110 ? e1 : -110) : 110;
      }
      eb = __builtin_amdgcn_readfirstlane(eb);
      e1 = __builtin_amdgcn_readfirstlane(e1);
      const float keep = __builtin_ldexpf(tot, e1 - eS), sx = pow2(e1);
      eS = e1;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[nt][pt][i] *= keep;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const f32x4 w0 = *(const f32x4*)(hs.w + 32 * kk + 4 * lg) * sx, w1 = *(const f32x4*)(hs.w + 32 * kk + 16 + 4 * lg) * sx;
        Split f[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = (float)xf[pt][2 * kk][i] * w0[i];
            v[4 + i] = (float)xf[pt][2 * kk + 1][i] * w1[i];
          }
          f[pt] = split8(v, one);
        }
        const uint16_t* br4 = bt + (32 * kk + 4 * lg + (lr >> 2)) * kPitchB + 4 * (lr & 3);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const f16x8 bf = join(read_transposed(br4 + 16 * nt), read_transposed(br4 + 16 * kPitchB + 16 * nt));
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) st[nt][pt] = mfma(bf, f[pt].hi, st[nt][pt]);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) st[nt][pt] = mfma(bf, f[pt].lo, st[nt][pt]);
        }
      }
    }
    if (ch + 1 < chunks) store_chunk(c0 + kChunk, par ^ 1);
    __syncthreads();
  }

  if (!OUT || len <= t1) {
    const float undo = pow2(-eS);
    const int64_t base = OUT ? slot * a.H + h : ((seg + 1) * a.batch + b) * a.H + h;
    float* dst = OUT ? a.state : sg.state;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
      if (pw + 16 * pt < cols) {
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
          *(f32x4*)(dst + (base * a.P + pc + pw + 16 * pt) * 128 + 16 * nt + 4 * lg) = st[nt][pt] * undo;
      }
    if (!OUT && live && scalars && pc == 0 && lane == 0) sg.decay[base] = __builtin_amdgcn_exp2f((float)seg_log);
  }
}

// The carries before each segment, of rows of more than one: a running fma over
// the segments' additions, four values a thread, all of a thread's loads in
// flight.
__global__ __launch_bounds__(256) void k_full_join(FullArgs a, Segments sg) {
  const int64_t b = blockIdx.y, i = (int64_t)blockIdx.x * 256 + threadIdx.x, per_row = a.H * a.P * 32;
  if (i >= per_row) return;
  const int64_t slot = full_slot(a, b), len = slot < 0 ? 0 : full_length(a, b);
  const int64_t started = (len + sg.tokens - 1) / sg.tokens;
  if (started < 2) return;
  const int64_t h = i / (a.P * 32);
  f32x4 cur = *(const f32x4*)(a.state + (slot * per_row + i) * 4);
  f32x4* at = (f32x4*)sg.state + b * per_row + i;
  const int64_t step = a.batch * per_row;
  at[0] = cur;
  for (int64_t q0 = 1; q0 < started; q0 += 8) {
    f32x4 v[8];
    float d[8];
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
        for (int e = 0; e < 4; ++e) cur[e] = __builtin_fmaf(cur[e], d[k], v[k][e]);
        at[(q0 + k) * step] = cur;
      }
  }
}

}  // namespace m2r

using namespace m2r;

namespace m2r {

// How many segments a call's tokens are split into.
Segments full_segments(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G) {
  const int64_t hpg = H / G, blocks = (hpg * ((P + 63) / 64) + 3) / 4, chunks = (L + kChunk - 1) / kChunk;
  const int64_t groups = blocks * G * batch;
  int64_t want = groups >= 192 ? 1 : 256 / groups;
  want = want < chunks ? want : chunks;
  const int64_t per = (chunks + want - 1) / want;
  return Segments{per * kChunk, (int)((chunks + per - 1) / per), nullptr, nullptr};
}

int64_t full_chunks_workspace(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G) {
  const Segments sg = full_segments(batch, L, H, P, G);
  return sg.count > 1 ? (int64_t)sg.count * batch * H * (P * 128 + 1) * 4 : 0;
}

hipError_t launch_full_chunks(const FullArgs& a, void* workspace, hipStream_t stream) {
  Segments sg = full_segments(a.batch, a.L, a.H, a.P, a.G);
  const int64_t hpg = a.H / a.G, blocks = (hpg * ((a.P + 63) / 64) + 3) / 4;
  if (sg.count > 1) {
    sg.state = (float*)workspace;
    sg.decay = sg.state + (int64_t)sg.count * a.batch * a.H * a.P * 128;
  }
  // 16-byte pieces through buffers: rows that do not overlap, and 64 of them
  // within 31-bit offsets
  const int64_t far = (int64_t)1 << 23, dense = a.H * a.P;
  const bool aligned = a.P % 8 == 0 && ((a.xs_b | a.xs_l | a.bs_b | a.bs_l | a.cs_b | a.cs_l) & 7) == 0 &&
                       (((uintptr_t)a.x | (uintptr_t)a.Bm | (uintptr_t)a.Cm | (uintptr_t)a.y) & 15) == 0 &&
                       a.xs_l >= dense && a.bs_l >= a.G * 128 && a.cs_l >= a.G * 128 && a.ds_l >= a.H &&
                       a.xs_l < far && a.bs_l < far && a.cs_l < far && a.ds_l < far;
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
