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
// pitch of 4 banks past a multiple of 64 puts them on all banks once), B and
// x as transposing reads of 4 rows by 32 bytes per 16 lanes (8 banks apart).
constexpr int kPitchC = 136, kPitchB = 144, kPitchX = 80;

struct ChunkShared {
  uint16_t c[kChunk * kPitchC];        // each 32 coordinates in the order of the carry's fragments
  uint16_t b[kChunk * kPitchB];
  uint16_t x[4][kChunk * kPitchX];
  u32x4 m[4][2][6][64];                // masked score fragments: high and low halves
  float lh[4][kChunk], ll[4][kChunk];  // l_t log2(e) as a sum of two binary32
  float dt[4][kChunk], w[4][kChunk], el[4][kChunk];
  float tot[4], wmax[4];
  int km[4][4];
  int bad[2];                          // a non-finite x in this chunk, by chunk parity
};

struct Segments {
  int64_t tokens;     // of a segment, a multiple of kChunk
  int count;
  // carries of rows that go on past their first segment, [count, batch, H, P,
  // 128]: 0 the row's first carry (the pool's own is overwritten by the last
  // segment while others still start), 1 the carry after segment 0, q > 1 what
  // segment q - 1 adds to a zero carry; and the decay over segment q - 1
  float* state;
  float* decay;       // [count, batch, H]
};

__device__ __forceinline__ float wave_max(float v) {   // of non-negative values; NaN is passed over
#define M2R_MAX_DPP(ctrl)                                                                                        \
  v = __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, \
                                                                              0xF, 0xF, true)))
  M2R_MAX_DPP(0xB1);
  M2R_MAX_DPP(0x4E);
  M2R_MAX_DPP(0x141);
  M2R_MAX_DPP(0x140);
#undef M2R_MAX_DPP
  const int iv = __builtin_bit_cast(int, v);
  const auto r = __builtin_amdgcn_permlane16_swap(iv, iv, false, false);
  v = __builtin_fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
  const int jv = __builtin_bit_cast(int, v);
  const auto q = __builtin_amdgcn_permlane32_swap(jv, jv, false, false);
  v = __builtin_fmaxf(__builtin_bit_cast(float, (int)q[0]), __builtin_bit_cast(float, (int)q[1]));
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
// floor(log2 v) of a positive normal v (-127 for zero and subnormals).
__device__ __forceinline__ int exponent_of(float v) { return ((__builtin_bit_cast(int, v) >> 23) & 255) - 127; }
__device__ __forceinline__ float pow2(int k) { return __builtin_ldexpf(1.0f, k); }

// v as the sum of two binary16, in units in which the largest value has the
// exponent 14: the first carries 11 bits, the second the next 11 (whatever is
// left above 2^-25), so that a product of a binary16 factor with both keeps
// 22 bits, and is summed in binary32 by the matrix instruction.
struct Split { f16x8 hi, lo; };
__device__ __forceinline__ Split split8(const float* v) {
  Split s;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 h = __builtin_convertvector((f32x2{v[j], v[j + 1]}), f16x2);
    const f16x2 l = __builtin_convertvector(
        (f32x2{__builtin_fmaf((float)h[0], -1.0f, v[j]), __builtin_fmaf((float)h[1], -1.0f, v[j + 1])}), f16x2);
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

template <bool ALIGNED>
__device__ __forceinline__ u32x4 load8(const uint16_t* p, int64_t valid) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (ALIGNED) {
    if (valid > 0) v = *(const u32x4*)p;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) v[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  }
  return v;
}

__device__ __forceinline__ double scan_add64(double v) {   // inclusive, over the wave
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const double o = __shfl_up(v, by);
    if (lane >= by) v += o;
  }
  return v;
}

// A workgroup steps four blocks of 64 columns (a head's channels) of one
// group, two waves each, over one segment of one batch row's tokens.  OUT:
// readouts and the pool's carry; else the segment's end for the segments
// after it.
template <bool ALIGNED, bool OUT>
__global__ __launch_bounds__(512, 2) void k_full_chunks(FullArgs a, Segments sg) {
  __shared__ ChunkShared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pair = wave >> 1, half = wave & 1;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t hpg = a.H / a.G, per_head = (a.P + 63) / 64, blocks = (hpg * per_head + 3) / 4;
  int64_t id = blockIdx.x;
  const int64_t blk = id % blocks;
  id /= blocks;
  const int64_t g = id % a.G;
  id /= a.G;
  const int64_t b = id % a.batch;
  const int64_t seg = id / a.batch;

  const int64_t slot = full_slot(a, b);
  const int64_t len = slot < 0 ? 0 : full_length(a, b);
  const int64_t t0 = seg * sg.tokens, t1 = t0 + sg.tokens < a.L ? t0 + sg.tokens : a.L;
  const int64_t n = len < t0 ? 0 : (len < t1 ? len : t1) - t0;   // the segment's tokens
  if (!OUT && len <= t1) return;                                   // no later segment reads this one

  // this pair's head and columns (idle past the group's last block)
  const int64_t unit = blk * 4 + pair;
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

  // the carry: S[16 nt + 4 lg + i][column] as s_[nt][pt][i], 2^-eS times its value
  f32x4 st[8][2];
  int eS = 0;
#pragma unroll
  for (int pt = 0; pt < 2; ++pt) {
    const int64_t p = pw + 16 * pt;
    const bool in = p < cols;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    auto row = [&](const float* base, int64_t at) { return base + ((at * a.H + h) * a.P + pc + p) * 128 + 4 * lg; };
    const int64_t per = a.batch;
    // the row's only segment, or the first of the states' pass: the pool's carry
    const bool from_pool = seg == 0 && (!OUT || len <= t1);
    const float* src = from_pool ? row(a.state, slot) : row(sg.state, (seg ? per : 0) + b);
    const bool read = in && (OUT || seg == 0);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) st[nt][pt] = read ? *(const f32x4*)(src + 16 * nt) : zero;
    if (!OUT && seg == 0 && in) {
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) *(f32x4*)(const_cast<float*>(row(sg.state, b)) + 16 * nt) = st[nt][pt];
    }
    if (OUT) {
      for (int64_t q = 2; q <= seg; ++q) {
        const float d = sg.decay[(q * per + b) * a.H + h];
        const float* add = row(sg.state, q * per + b);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const f32x4 v = in ? *(const f32x4*)(add + 16 * nt) : zero;
#pragma unroll
          for (int i = 0; i < 4; ++i) st[nt][pt][i] = __builtin_fmaf(st[nt][pt][i], d, v[i]);
        }
      }
    }
  }
  const float av = a.A[h], dh = load_param(a.D, a.d_f32, (int)h), bias = load_param(a.dt_bias, a.db_f32, (int)h);
  double seg_log = 0.0;   // the segment's decay so far, as a power of two

  // global loads of a chunk: B and C two, x four 16-byte pieces a thread
  u32x4 rb[2], rc[2], rx[4];
  uint16_t rdt = 0;
  const uint16_t *bp = a.Bm + b * a.bs_b + g * 128, *cp = a.Cm + b * a.cs_b + g * 128;
  auto load_chunk = [&](int64_t c0) {   // tokens t0 + c0 ...
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = k * 512 + tid, r = i >> 4, part = i & 15;
      const bool in = c0 + r < n;
      rb[k] = load8<ALIGNED>(bp + (t0 + c0 + r) * a.bs_l + 8 * part, in ? 8 : 0);
      if (OUT) rc[k] = load8<ALIGNED>(cp + (t0 + c0 + r) * a.cs_l + 8 * part, in ? 8 : 0);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {   // the pair's own columns: 128 threads, 64 rows of 8 pieces
      const int i = k * 128 + half * 64 + lane, r = i >> 3, part = i & 7;
      const int64_t left = c0 + r < n ? cols - 8 * part : 0;
      rx[k] = load8<ALIGNED>(a.x + b * a.xs_b + (t0 + c0 + r) * a.xs_l + h * a.P + pc + 8 * part, left);
    }
    if (half == 0) rdt = c0 + lane < n ? a.dt[b * a.ds_b + (t0 + c0 + lane) * a.ds_l + h] : 0;
  };
  if (tid < 2) s.bad[tid] = 0;
  load_chunk(0);
  __syncthreads();

  const int64_t chunks = (n + kChunk - 1) / kChunk;
  for (int64_t ch = 0; ch < chunks; ++ch) {
    const int64_t c0 = ch * kChunk;
    const int par = (int)(ch & 1);
    // ---- the chunk into LDS
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = k * 512 + tid, r = i >> 4, part = i & 15;
      *(u32x4*)(s.b + r * kPitchB + 8 * part) = rb[k];
      if (OUT) {
        // coordinates 32 kk + 16 T + 4 q + i of a row stand at 32 kk + 8 q + 4 T + i
        const int kk = part >> 2, T = (part >> 1) & 1, q = 2 * (part & 1);
        uint16_t* d = s.c + r * kPitchC + 32 * kk + 8 * q + 4 * T;
        *(u32x2*)d = u32x2{rc[k][0], rc[k][1]};
        *(u32x2*)(d + 8) = u32x2{rc[k][2], rc[k][3]};
      }
    }
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * 128 + half * 64 + lane, r = i >> 3, part = i & 7;
      *(u32x4*)(s.x[pair] + r * kPitchX + 8 * part) = rx[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= ((rx[k][j] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;   // exponent 31
    }
    if (OUT && odd) s.bad[par] = 1;
    if (tid == 0) s.bad[par ^ 1] = 0;
    if (half == 0) {   // lane = token
      const bool in = c0 + lane < n;
      const float dt = in ? full_dt(h2f(rdt) + bias) : 0.f;
      const double l = scan_add64((double)av * (double)dt * 1.4426950408889634);
      const double last = __shfl(l, 63);
      const float lh = (float)l;
      const float w = dt * __builtin_amdgcn_exp2f((float)(last - l));
      s.lh[pair][lane] = lh;
      s.ll[pair][lane] = __builtin_fabsf(lh) < __builtin_inff() ? (float)(l - (double)lh) : 0.f;
      s.dt[pair][lane] = dt;
      s.w[pair][lane] = w;
      s.el[pair][lane] = __builtin_amdgcn_exp2f(lh);
      const float wm = wave_max(w);
      if (lane == 0) {
        s.tot[pair] = __builtin_amdgcn_exp2f((float)last);
        s.wmax[pair] = wm;
      }
      seg_log += last;
    }
    __syncthreads();
    if (ch + 1 < chunks) load_chunk(c0 + kChunk);

    const uint16_t* xt = s.x[pair];
    if (OUT && s.bad[par]) {
      // A non-finite x must not reach earlier tokens, which the matrix
      // products would let it do (0 * inf): this chunk token by token.
      const float undo = pow2(-eS);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) st[nt][pt] *= undo;
      eS = 0;
      const int64_t left = n - c0 < kChunk ? n - c0 : kChunk;
      for (int t = 0; t < left; ++t) {
        const float dt = s.dt[pair][t];
        const float decay = __builtin_amdgcn_exp2f(
            t ? (s.lh[pair][t] - s.lh[pair][t - 1]) + (s.ll[pair][t] - s.ll[pair][t - 1]) : s.lh[pair][0]);
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          const float xv = h2f(xt[t * kPitchX + pw + 16 * pt]), in = xv * dt;
          float acc = 0.f;
#pragma unroll
          for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float bv = h2f(s.b[t * kPitchB + 16 * nt + 4 * lg + i]);
              const float cv = h2f(s.c[t * kPitchC + 32 * (nt >> 1) + 8 * lg + 4 * (nt & 1) + i]);
              st[nt][pt][i] = __builtin_fmaf(st[nt][pt][i], decay, in * bv);
              acc = __builtin_fmaf(st[nt][pt][i], cv, acc);
            }
          acc = butterfly_add<5>(butterfly_add<4>(acc));
          if (lg == 0 && pw + 16 * pt < cols)
            a.y[((b * a.L + t0 + c0 + t) * a.H + h) * a.P + pc + pw + 16 * pt] = f2h(__builtin_fmaf(xv, dh, acc));
        }
      }
      __syncthreads();
      continue;
    }

    // x fragments: tokens 16 T + 4 lg + r of column pw + 16 pt
    f16x4 xf[2][4];
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int T = 0; T < 4; ++T)
        xf[pt][T] = read_transposed(xt + (16 * T + 4 * lg + (lr >> 2)) * kPitchX + 32 * half + 16 * pt + 4 * (lr & 3));

    float smax = 0.f;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int i = 0; i < 4; ++i) smax = __builtin_fmaxf(smax, __builtin_fabsf(st[nt][pt][i]));
    smax = wave_max(smax);
    if (!(smax < __builtin_inff())) {   // an infinite channel must not set the others' scale
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
    }

    if constexpr (OUT) {
      // ---- masked scores of this wave's two row tiles (of 16 tokens)
      auto scores = [&](auto tile) {
        constexpr int I = decltype(tile)::value;
        f16x8 cf[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) cf[kk] = *(const f16x8*)(s.c + (16 * I + lr) * kPitchC + 32 * kk + 8 * lg);
        const float th = s.lh[pair][16 * I + lr], tl = s.ll[pair][16 * I + lr];
        float v[16];
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j <= I; ++j) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint16_t* r = s.b + (16 * j + lr) * kPitchB + 32 * kk + 4 * lg;
            acc = mfma(join(*(const f16x4*)r, *(const f16x4*)(r + 16)), cf[kk], acc);
          }
          const f32x4 sh = *(const f32x4*)(s.lh[pair] + 16 * j + 4 * lg), sl = *(const f32x4*)(s.ll[pair] + 16 * j + 4 * lg);
          const f32x4 sd = *(const f32x4*)(s.dt[pair] + 16 * j + 4 * lg);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f((th - sh[i]) + (tl - sl[i]));
            float m = (acc[i] * sd[i]) * e;
            if (j == I) m = 4 * lg + i <= lr ? m : 0.f;
            v[4 * j + i] = m;
            mx = __builtin_fmaxf(mx, __builtin_fabsf(m));
          }
        }
        mx = wave_max(mx);
        if (!(mx < __builtin_inff())) {
          mx = 0.f;
#pragma unroll
          for (int i = 0; i < 4 * I + 4; ++i) {
            const float q = __builtin_fabsf(v[i]);
            mx = __builtin_fmaxf(mx, q < __builtin_inff() ? q : 0.f);
          }
          mx = wave_max(mx);
        }
        int km = 14 - exponent_of(mx);
        km = km > 40 ? 40 : km;   // below 2^-25 a score times any x is nothing in the readout
        const float scale = pow2(km);
        if (lane == 0) s.km[pair][I] = km;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < 4 * I + 4 ? v[i] * scale : 0.f;
#pragma unroll
        for (int kk = 0; kk <= I / 2; ++kk) {
          const Split f = split8(v + 8 * kk);
          constexpr int base = I < 2 ? I : 2 * I - 2;
          s.m[pair][0][base + kk][lane] = __builtin_bit_cast(u32x4, f.hi);
          s.m[pair][1][base + kk][lane] = __builtin_bit_cast(u32x4, f.lo);
        }
      };
      if (half == 0) {
        scores(std::integral_constant<int, 0>{});
        scores(std::integral_constant<int, 3>{});
      } else {
        scores(std::integral_constant<int, 1>{});
        scores(std::integral_constant<int, 2>{});
      }

      // ---- S C_t: rows = columns of x, columns = tokens
      int kS = 14 - exponent_of(smax);
      kS = kS > 120 ? 120 : kS;
      const float ss = pow2(kS);
      f32x4 acc[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) acc[i][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        Split f[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = st[2 * kk + (i >> 2)][pt][i & 3] * ss;
          f[pt] = split8(v);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x8 cf = *(const f16x8*)(s.c + (16 * i + lr) * kPitchC + 32 * kk + 8 * lg);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            acc[i][pt] = mfma(f[pt].hi, cf, acc[i][pt]);
            acc[i][pt] = mfma(f[pt].lo, cf, acc[i][pt]);
          }
        }
      }
      __syncthreads();   // both waves' score fragments are there
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int km = s.km[pair][i];
        const float f = __builtin_ldexpf(s.el[pair][16 * i + lr], km - kS - eS);
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][pt][r] *= f;
        }
#pragma unroll
        for (int kk = 0; kk <= i / 2; ++kk) {
          const int at = (i < 2 ? i : 2 * i - 2) + kk;
          const f16x8 mh = __builtin_bit_cast(f16x8, s.m[pair][0][at][lane]);
          const f16x8 ml = __builtin_bit_cast(f16x8, s.m[pair][1][at][lane]);
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            const f16x8 xx = join(xf[pt][2 * kk], xf[pt][2 * kk + 1]);
            acc[i][pt] = mfma(xx, mh, acc[i][pt]);
            acc[i][pt] = mfma(xx, ml, acc[i][pt]);
          }
        }
        const float back = pow2(-km);
        const int64_t t = c0 + 16 * i + lr;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          const int p = 32 * half + 16 * pt + 4 * lg;
          const f16x4 xv = *(const f16x4*)(xt + (16 * i + lr) * kPitchX + p);
          f16x4 out;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = __builtin_fmaf((float)xv[r], dh, acc[i][pt][r] * back);
            asm volatile("" : "+v"(v));   // rounded to binary32 first in every instance
            out[r] = (_Float16)v;
          }
          if (t < n) {
            uint16_t* yp = a.y + ((b * a.L + t0 + t) * a.H + h) * a.P + pc + p;
            if constexpr (ALIGNED) {
              if (p < cols) *(f16x4*)yp = out;
            } else {
              const s16x4v bits = __builtin_bit_cast(s16x4v, out);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (p + r < cols) yp[r] = (uint16_t)bits[r];
            }
          }
        }
      }
    }

    // ---- the carry after the chunk
    {
      uint32_t xm = 0;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int T = 0; T < 4; ++T) {
          const u32x2 q = __builtin_bit_cast(u32x2, xf[pt][T]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t lo = q[j] & 0x7fffu, hi = (q[j] >> 16) & 0x7fffu;
            xm = xm > lo ? xm : lo;
            xm = xm > hi ? xm : hi;
          }
        }
      const float xmax = wave_max(xm >= 0x7c00u ? 65536.0f : h2f((uint16_t)xm)), wmax = s.wmax[pair];
      // x w 2^kX below 2^15, unless the carry would leave binary32
      int kX = eS;
      if (xmax > 0.f && wmax > 0.f && wmax < __builtin_inff()) {
        kX = 13 - exponent_of(xmax) - exponent_of(wmax);
        const int room = eS + (100 - exponent_of(smax) < 120 ? 100 - exponent_of(smax) : 120);
        kX = kX < room ? kX : room;
        kX = kX < 120 ? (kX > -120 ? kX : -120) : 120;
      }
      const float keep = __builtin_ldexpf(s.tot[pair], kX - eS), sx = pow2(kX);
      eS = kX;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[nt][pt][i] *= keep;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const f32x4 w0 = *(const f32x4*)(s.w[pair] + 32 * kk + 4 * lg), w1 = *(const f32x4*)(s.w[pair] + 32 * kk + 16 + 4 * lg);
        Split f[2];
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = (float)xf[pt][2 * kk][i] * (w0[i] * sx);
            v[4 + i] = (float)xf[pt][2 * kk + 1][i] * (w1[i] * sx);
          }
          f[pt] = split8(v);
        }
        const uint16_t* bt = s.b + (32 * kk + 4 * lg + (lr >> 2)) * kPitchB + 4 * (lr & 3);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const f16x8 bf = join(read_transposed(bt + 16 * nt), read_transposed(bt + 16 * kPitchB + 16 * nt));
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            st[nt][pt] = mfma(bf, f[pt].hi, st[nt][pt]);
            st[nt][pt] = mfma(bf, f[pt].lo, st[nt][pt]);
          }
        }
      }
    }
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
    if (!OUT && live && half == 0 && pc == 0 && lane == 0) sg.decay[base] = __builtin_amdgcn_exp2f((float)seg_log);
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
  const int64_t hpg = a.H / a.G, blocks = (hpg * ((a.P + 63) / 64) + 3) / 4, groups = blocks * a.G * a.batch;
  if (sg.count > 1) {
    sg.state = (float*)workspace;
    sg.decay = sg.state + (int64_t)sg.count * a.batch * a.H * a.P * 128;
  }
  const bool aligned = a.P % 8 == 0 && ((a.xs_b | a.xs_l | a.bs_b | a.bs_l | a.cs_b | a.cs_l) & 7) == 0 &&
                       (((uintptr_t)a.x | (uintptr_t)a.Bm | (uintptr_t)a.Cm | (uintptr_t)a.y) & 15) == 0;
  if (groups * sg.count > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 block(512);
  if (sg.count > 1) {
    const dim3 grid((unsigned)(groups * (sg.count - 1)));
    if (aligned) hipLaunchKernelGGL((k_full_chunks<true, false>), grid, block, 0, stream, a, sg);
    else hipLaunchKernelGGL((k_full_chunks<false, false>), grid, block, 0, stream, a, sg);
  }
  const dim3 grid((unsigned)(groups * sg.count));
  if (aligned) hipLaunchKernelGGL((k_full_chunks<true, true>), grid, block, 0, stream, a, sg);
  else hipLaunchKernelGGL((k_full_chunks<false, true>), grid, block, 0, stream, a, sg);
  return hipGetLastError();
}

}  // namespace m2r
