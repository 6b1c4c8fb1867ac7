// Low-rank adapters of many requests beside a shared projection, for gfx950:
//   out[m] = half(base[m] + scale[a] up[a] (down[a] x[m])),  a = ids[m],
// and out[m] = base[m] where ids[m] names no adapter (negative, or not below
// the number of adapters).  x [M, K], base and out [M, N] binary16 rows,
// down [n, r, Kp], up [n, N, r] binary16, scale [n] binary32; r the rank and
// Kp = K, each rounded up to 8, the rest zeros.
//
// Two launches on the matrix cores, rows in tiles of 16.  The first forms the
// hidden values down x of a tile over a slice of K, in binary32; the second
// adds the slices up and multiplies by up.  The rows of a tile that share an
// adapter are one product, whose other columns are computed and dropped: a
// prompt's rows are mostly one such group, a decode step's rows one each.
//
// Bound by memory and by the latency of a short chain of loads (ids, weights
// and rows, hidden values): 2 r (K + N) operations for 2 (K + 2 N) bytes a row.
// 2,500 rows of rank 32 over K = 4,096, N = 18,560 (six adapters): 72 us, the
// first launch 15 and the second 46 warm, 215 MB at 3.0 TB/s, where a copy of
// base to out alone takes 38.  64 rows of 48 adapters of rank 16, K = 8,192,
// N = 4,096: 14 us; one row, K = 4,096, N = 18,560: 8 us, two launches.
#include "m2r_device.h"
#include "m2r_abi_util.h"
#include "m2r_tile.h"

#include <initializer_list>

namespace m2r {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t h16x8 __attribute__((ext_vector_type(8)));

struct AdapterArgs {
  const uint16_t* x;
  int64_t xs;
  const uint16_t* base;
  int64_t bs;
  const uint16_t *down, *up;
  const float* scale;
  const int32_t* ids;
  uint16_t* out;
  int64_t os;
  float* hidden;        // [slices, M, r]
  int64_t M, K, Kp, N, n;
  int r;
  int rank;             // r - 7 ... r: a hidden value past it counts as 0, whatever x holds
  int slices;           // of K, `slice` long each (a multiple of 64)
  int64_t slice;
  int members;          // workgroups (waves in the second launch) among which a tile's groups are dealt, a power of two to 16
  int64_t span;         // outputs of a wave in the second launch, a multiple of 64
  uint32_t spans;
};

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// 8 binary16 values at p (2-byte aligned), zeros from `valid` on.
__device__ __forceinline__ f16x8 load_f16x8(const uint16_t* p, int64_t valid) {
  h16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (valid >= 8) __builtin_memcpy(&v, p, 16);
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) v[j] = p[j];
  }
  return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ h16x8 load_h16x8(const uint16_t* p) {   // all 8, without a branch
  h16x8 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// Ranks at ... at + 7 of a row of `up`, zeros from r on.
__device__ __forceinline__ f16x8 load_ranks(const uint16_t* row, int at, int r) {
  const h16x8 v = load_h16x8(row + (at < r ? at : 0));
  const h16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
  return __builtin_bit_cast(f16x8, at < r ? v : zero);
}
// The adapter of row m; -1 for none and past the last row.
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int64_t m) {
  const int id = m < a.M ? a.ids[m] : -1;
  return id >= 0 && id < a.n ? id : -1;
}

// Of 16 members each takes the group whose first row it is, without counting
// the groups before it: leaves that group in `rows`, the tile's, or nothing.
__device__ __forceinline__ int only_group(int id, int member, uint32_t& rows) {
  const uint32_t group = (uint32_t)__ballot(id == __builtin_amdgcn_readlane(id, member)) & rows;
  rows = (group >> member & 1) && !(group & ((1u << member) - 1)) ? group : 0;
  return member;
}

// One wave per (tile, slice of K / 4): its four quarters meet in LDS.  (More
// loads in flight at a time, three to six steps', changed nothing.)
// RT: 16-rank tiles at a time.  MT: row tiles.
template <int RT, int MT>
__global__ __launch_bounds__(256) void k_adapter_down(AdapterArgs a) {
  __shared__ f32x4 part[3][MT * RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  uint32_t w = blockIdx.x;   // (64-bit divisions here would take a microsecond)
  const int member = (int)(w % (uint32_t)a.members);
  w /= (uint32_t)a.members;
  const int slice = (int)(w % (uint32_t)a.slices);
  const int64_t m0 = (int64_t)(w / (uint32_t)a.slices) * (16 * MT);
  int id[MT];
  uint32_t todo = 0;
  const uint16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + 16 * i + lr;
    id[i] = adapter_of(a, m);
    todo |= ((uint32_t)__ballot(id[i] >= 0) & 0xffffu) << (16 * i);
    xr[i] = a.x + (m < a.M ? m : a.M - 1) * a.xs;
  }
  int group = 0;
  if (MT == 1 && a.members == 16) group = only_group(id[0], member, todo);
  const int64_t quarter = (a.slice / 64 + 3) / 4 * 64;
  const int64_t s1 = (slice + 1) * a.slice < a.Kp ? (slice + 1) * a.slice : a.Kp;
  const int64_t k0 = slice * a.slice + wave * quarter, k1 = k0 + quarter < s1 ? k0 + quarter : s1;
  for (; todo; ++group) {
    const int first = __builtin_ctz(todo);
    int cur = 0;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (first >> 4 == i) cur = __builtin_amdgcn_readlane(id[i], first & 15);
#pragma unroll
    for (int i = 0; i < MT; ++i) todo &= ~(((uint32_t)__ballot(id[i] == cur) & 0xffffu) << (16 * i));
    if (MT == 1 && (group & (a.members - 1)) != member) continue;
    for (int r0 = 0; r0 < a.r; r0 += 16 * RT) {
      f32x4 acc[MT][RT];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint16_t* dr[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {   // ranks past the last read its row and are not stored
        const int j = r0 + 16 * t + lr;
        dr[t] = a.down + ((int64_t)cur * a.r + (j < a.r ? j : a.r - 1)) * a.Kp;
      }
      // 64 inputs at a time in two products, the lane's 16 of them neighbours:
      // the pair of loads covers whole 128-byte lines of a row
#pragma unroll 2
      for (int64_t kb = k0; kb < k1; kb += 64) {
        f16x8 xv[2][MT], dv[2][RT];
        if (kb + 64 <= k1 && kb + 64 <= a.K) {   // (one answer for the wave)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int64_t k = kb + 16 * lg + 8 * u;
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[u][i] = __builtin_bit_cast(f16x8, load_h16x8(xr[i] + k));
#pragma unroll
            for (int t = 0; t < RT; ++t) dv[u][t] = __builtin_bit_cast(f16x8, load_h16x8(dr[t] + k));
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int64_t k = kb + 16 * lg + 8 * u;
            const bool in = k < k1;
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[u][i] = load_f16x8(xr[i] + k, in ? a.K - k : 0);
#pragma unroll
            for (int t = 0; t < RT; ++t) dv[u][t] = load_f16x8(dr[t] + k, in ? 8 : 0);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[i][t] = mfma16(dv[u][t], xv[u][i], acc[i][t]);
      }
      __syncthreads();
      if (wave) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < RT; ++t) part[wave - 1][i * RT + t][lane] = acc[i][t];
      }
      __syncthreads();
      if (wave == 0) {   // columns = rows m, rows = ranks 4 lg ...
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int64_t m = m0 + 16 * i + lr;
          if (id[i] == cur && m < a.M) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              f32x4 v = acc[i][t];
#pragma unroll
              for (int q = 0; q < 3; ++q) v += part[q][i * RT + t][lane];
              const int j = r0 + 16 * t + 4 * lg;
              if (j < a.r) *(f32x4*)(a.hidden + (slice * a.M + m) * a.r + j) = v;
            }
          }
        }
      }
    }
  }
}

// v 2^k as the sum of two binary16: 22 bits of the product's operand (and nothing
// below 2^-39 of the row's largest), where one alone would round the hidden
// values to 11.  An infinity's second part is 0.
__device__ __forceinline__ void split_f16(const float* v, float scale, f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 h = __builtin_convertvector((f32x2{v[j] * scale, v[j + 1] * scale}), f16x2);
    const float r0 = __builtin_fmaf(v[j], scale, -(float)h[0]), r1 = __builtin_fmaf(v[j + 1], scale, -(float)h[1]);
    const f16x2 l = __builtin_convertvector(
        (f32x2{__builtin_isinf(v[j]) ? 0.f : r0, __builtin_isinf(v[j + 1]) ? 0.f : r1}), f16x2);
    hi[j] = h[0];
    hi[j + 1] = h[1];
    lo[j] = l[0];
    lo[j + 1] = l[1];
  }
}

// The hidden values of row m (where `mine`) in the layout of a product's
// columns, times 2^k as two binary16; returns 2^-k.
template <int KS>
__device__ __forceinline__ float hidden_fragments(const AdapterArgs& a, int64_t m, bool mine, float sc, f16x8* hi, f16x8* lo) {
  const int lg = (threadIdx.x & 63) >> 4;
  float v[KS][8], mx = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    const int j0 = 32 * k + 8 * lg;
    if (mine && j0 < a.r) {
      const float* h = a.hidden + m * a.r + j0;
      for (int q = 0; q < a.slices; ++q) {
        const f32x4 u0 = *(const f32x4*)(h + (int64_t)q * a.M * a.r), u1 = *(const f32x4*)(h + (int64_t)q * a.M * a.r + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[k][j] += u0[j];
          v[k][4 + j] += u1[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[k][j] = j0 + j < a.rank ? v[k][j] * sc : 0.f;
        mx = __builtin_fmaxf(mx, __builtin_fabsf(v[k][j]));
      }
    }
  }
  // the row's largest, over its four lanes
  const int iv = __builtin_bit_cast(int, mx);
  const auto p = __builtin_amdgcn_permlane16_swap(iv, iv, false, false);
  mx = __builtin_fmaxf(__builtin_bit_cast(float, (int)p[0]), __builtin_bit_cast(float, (int)p[1]));
  const int jv = __builtin_bit_cast(int, mx);
  const auto q = __builtin_amdgcn_permlane32_swap(jv, jv, false, false);
  mx = __builtin_fmaxf(__builtin_bit_cast(float, (int)q[0]), __builtin_bit_cast(float, (int)q[1]));
  int e = 14 - (((__builtin_bit_cast(int, mx) >> 23) & 255) - 127);   // the largest below 2^15
  e = e > 100 ? 100 : e;
  const float up = __builtin_ldexpf(1.0f, e);
#pragma unroll
  for (int k = 0; k < KS; ++k) split_f16(v[k], up, hi[k], lo[k]);
  return __builtin_ldexpf(1.0f, -e);
}

// One wave per (MT tiles of 16 rows, span of outputs).  A lane holds row
// 16 i + lr of each tile and 8 neighbouring outputs of 32: output tile T of
// NT takes outputs 4 NT q + 4 T + k of the 16 NT as its rows 4 q + k.  The
// hidden values go in as two binary16, scaled by each row's largest.
// KS: 32-rank steps.  Two tiles of rows share the loads of `up` where rows are
// many (one at a time: 81 us for 76), and take 64 outputs at a time, whole
// 128-byte lines (32: 80 us for 76); few rows take 32, for more waves (64 rows:
// 15.8 us for 17.9).  Turning the products in LDS for rows of full lines cost
// more than the lines saved (82 us for 80).
template <int MT, int KS, int NT>
__global__ __launch_bounds__(256, KS == 1 ? 3 : 1) void k_adapter_up(AdapterArgs a) {
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t span = w % a.spans;
  w /= a.spans;
  const int member = (int)(w % (uint32_t)a.members);
  const int64_t m0 = (int64_t)(w / (uint32_t)a.members) * (16 * MT);
  if (m0 >= a.M) return;
  const int64_t n0 = span * a.span, n1 = n0 + a.span < a.N ? n0 + a.span : a.N;
  int id[MT];
  uint64_t todo = 0;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + 16 * i + lr;
    id[i] = adapter_of(a, m);
    todo |= (__ballot(m < a.M) & 0xffffull) << (16 * i);
  }
  int group = 0;
  if (MT == 1 && a.members == 16) {
    uint32_t rows = (uint32_t)todo;
    group = only_group(id[0], member, rows);
    todo = rows;
  }
  for (; todo; ++group) {
    const int first = __builtin_ctzll(todo);
    int cur = 0;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (first >> 4 == i) cur = __builtin_amdgcn_readlane(id[i], first & 15);
    bool mine[MT];
    const uint16_t* br[MT];
    uint16_t* orow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + 16 * i + lr;
      mine[i] = id[i] == cur && m < a.M;
      todo &= ~((__ballot(mine[i]) & 0xffffull) << (16 * i));
      br[i] = a.base + (m < a.M ? m : 0) * a.bs;
      orow[i] = a.out + (m < a.M ? m : 0) * a.os;
    }
    if (MT == 1 && (group & (a.members - 1)) != member) continue;
    if (cur < 0) {   // rows without an adapter
      for (int64_t n = n0 + 8 * lg; n < n1; n += 32)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          if (mine[i]) {
            if (n + 8 <= a.N) __builtin_memcpy(orow[i] + n, br[i] + n, 16);
            else
              for (int j = 0; j < 8; ++j)
                if (n + j < a.N) orow[i][n + j] = br[i][n + j];
          }
      continue;
    }
    f16x8 hi[MT][KS], lo[MT][KS];
    float back[MT];
    const float sc = a.scale[cur];
#pragma unroll
    for (int i = 0; i < MT; ++i) back[i] = hidden_fragments<KS>(a, m0 + 16 * i + lr, mine[i], sc, hi[i], lo[i]);
    const uint16_t* ub = a.up + (int64_t)cur * a.N * a.r;
    // the next step's base is on its way while this one is formed; `up` comes
    // from the L2, and a second set of its registers would cost a wave a SIMD
    h16x8 bv[MT][NT / 2], bn[MT][NT / 2];
    auto fetch = [&](int64_t nb, h16x8 (&bd)[MT][NT / 2]) {
      const int64_t n = nb + 4 * NT * lg;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int u = 0; u < NT / 2; ++u)
          bd[i][u] = nb + 16 * NT <= a.N ? load_h16x8(br[i] + n + 8 * u)
                                         : __builtin_bit_cast(h16x8, load_f16x8(br[i] + n + 8 * u, a.N - n - 8 * u));
    };
    fetch(n0, bv);
    for (int64_t nb = n0; nb < n1; nb += 16 * NT) {
      f16x8 uf[NT][KS];
#pragma unroll
      for (int T = 0; T < NT; ++T) {
        const int64_t row = nb + 4 * NT * (lr >> 2) + 4 * T + (lr & 3);
        const uint16_t* ur = ub + (row < a.N ? row : a.N - 1) * a.r;
#pragma unroll
        for (int k = 0; k < KS; ++k) uf[T][k] = load_ranks(ur, 32 * k + 8 * lg, a.r);
      }
      // (behind the loads of `up`, which are waited for first)
      if (nb + 16 * NT < n1) fetch(nb + 16 * NT, bn);
      f32x4 acc[MT][NT];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int T = 0; T < NT; ++T) acc[i][T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int T = 0; T < NT; ++T)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][T] = mfma16(uf[T][k], hi[i][k], acc[i][T]);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][T] = mfma16(uf[T][k], lo[i][k], acc[i][T]);
        }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        if (mine[i])
#pragma unroll
          for (int u = 0; u < NT / 2; ++u) {
            const int64_t n = nb + 4 * NT * lg + 8 * u;
            h16x8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              o[j] = f2h(__builtin_fmaf(acc[i][2 * u + (j >> 2)][j & 3], back[i], h2f(bv[i][u][j])));
            if (n + 8 <= a.N) __builtin_memcpy(orow[i] + n, &o, 16);
            else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < a.N) orow[i][n + j] = o[j];
            }
          }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int u = 0; u < NT / 2; ++u) bv[i][u] = bn[i][u];
    }
  }
}

constexpr int64_t kMemberRows = 512;
// Workgroups among which a tile's groups are dealt: few rows leave the chip idle
// otherwise, and of many rows most find no group of theirs.  us a call at rank
// 16, K = N = 4,096, 8 adapters, with 16 / 4 / 1 of them: 64 rows of 64 requests
// 10.8 / 14.7 / -, of two 10.7 / 9.2 / -; 128 rows of 128 15.3 / 15.7 / -, of
// two 14.2 / 9.5 / -; 256 rows of 256 19.8 / 18.9 / 49, of six 20.5 / 11.6 /
// 16.7; 512 rows of 512 31 / 28 / 50, of six 34 / 15.4 / 20.3; 1,024 rows of
// 1,024 54 / 41 / 57, of six 49 / 24.5 / 20.8.
static int adapter_members(int64_t M) {
  const int most = M <= 64 ? 16 : (M <= kMemberRows ? 4 : 1);
  int members = 1;
  while (members < most && members < M) members *= 2;
  return members;
}
// From here on two tiles share the loads of `down` in the first launch.  us a
// call with one / two, K = N = 4,096: 2,500 rows of rank 32, N = 18,560, 72 /
// 75; 8,000 rows of rank 16 60 / 57, of rank 128 199 / 169.
constexpr int64_t kPairRows = 4096;
// Waves to aim for in the second launch (2,500 rows of rank 32, N = 18,560: 4,096
// and 6,144 waves 1 to 2 us slower, 3,072 by 11).
constexpr int64_t kSpanWaves = 8192;

static void adapter_plan(AdapterArgs& a) {
  const int64_t tiles = (a.M + 15) / 16;
  a.members = adapter_members(a.M);
  // Slices of K for about 512 workgroups, of at least 512 each and at most four,
  // since the second launch adds them up for each span.
  int64_t s = 512 / (a.M > kPairRows ? (tiles + 1) / 2 : tiles * a.members);
  const int64_t most = (a.Kp + 511) / 512;
  s = s < most ? s : most;
  s = s < 1 ? 1 : (s > 4 ? 4 : s);
  a.slice = ((a.Kp + s - 1) / s + 63) / 64 * 64;
  a.slices = (int)((a.Kp + a.slice - 1) / a.slice);
}

}  // namespace m2r

using namespace m2r;

extern "C" int64_t m2r_adapters_workspace(int64_t M, int64_t K, int64_t N, int64_t r) {
  if (M <= 0 || K <= 0 || N <= 0 || r <= 0) return 0;
  AdapterArgs a{};
  a.M = M;
  a.Kp = (K + 7) / 8 * 8;
  adapter_plan(a);
  return 4 * a.slices * M * ((r + 7) / 8 * 8);
}

extern "C" int m2r_adapters_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride,
                                const void* down, const void* up, const float* scale, const int32_t* ids, void* out,
                                int64_t out_stride, int64_t M, int64_t K, int64_t N, int64_t adapters, int64_t rank,
                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M <= 0 || K <= 0 || N <= 0 || adapters <= 0 || rank <= 0) return m2r_fail("adapters: non-positive shape");
  const int64_t lim = (int64_t)1 << 24;
  if (M > lim || K > lim || N > lim || adapters > lim || rank > 256) return m2r_fail("adapters: size limits");
  for (const void* p : {x, base, down, up, (const void*)scale, (const void*)ids, (const void*)out, (const void*)workspace})
    if (!p) return m2r_fail("adapters: null pointer");
  if (((uintptr_t)down | (uintptr_t)up) & 15) return m2r_fail("adapters: down and up must be 16-byte aligned");
  if (x_stride < K || base_stride < N || out_stride < N) return m2r_fail("adapters: rows overlap");
  if ((uintptr_t)workspace & 15 || workspace_bytes < m2r_adapters_workspace(M, K, N, rank))
    return m2r_fail("adapters: workspace too small or not 16-byte aligned");
  AdapterArgs a{(const uint16_t*)x, x_stride, (const uint16_t*)base, base_stride, (const uint16_t*)down,
                (const uint16_t*)up, scale, ids, (uint16_t*)out, out_stride, (float*)workspace, M, K, (K + 7) / 8 * 8, N,
                adapters, (int)((rank + 7) / 8 * 8), (int)rank};
  adapter_plan(a);
  const int64_t tiles = (M + 15) / 16;
  if (tiles * a.members * a.slices > 0x7fffffff) return m2r_fail("adapters: grid limits exceeded");
  const bool pairs = M > kPairRows;
  const dim3 down_grid((unsigned)((pairs ? (tiles + 1) / 2 : tiles * a.members) * a.slices)), block(256);
  if (pairs) {
    if (rank <= 16) hipLaunchKernelGGL((k_adapter_down<1, 2>), down_grid, block, 0, stream, a);
    else if (rank <= 32) hipLaunchKernelGGL((k_adapter_down<2, 2>), down_grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_adapter_down<4, 2>), down_grid, block, 0, stream, a);
  } else {
    if (rank <= 16) hipLaunchKernelGGL((k_adapter_down<1, 1>), down_grid, block, 0, stream, a);
    else if (rank <= 32) hipLaunchKernelGGL((k_adapter_down<2, 1>), down_grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_adapter_down<4, 1>), down_grid, block, 0, stream, a);
  }
  int rc = m2r_check(hipGetLastError(), "adapters down launch");
  if (rc) return rc;
  // Two tiles share a pass over `up` where rows are many and the rank leaves
  // registers for both (2,048 rows of rank 128: 90 us with one, 107 with two).
  const bool wide = M > kMemberRows && rank <= 64;
  const int64_t groups = wide ? (M + 31) / 32 : tiles * a.members;
  int64_t spans = kSpanWaves / groups;
  const int64_t most = (N + 63) / 64;
  spans = spans < 1 ? 1 : (spans < most ? spans : most);
  a.span = ((N + spans - 1) / spans + 63) / 64 * 64;
  spans = (N + a.span - 1) / a.span;
  if (groups * spans > 0x7fffffff) return m2r_fail("adapters: grid limits exceeded");
  a.spans = (uint32_t)spans;
  const dim3 up_grid((unsigned)((groups * spans + 3) / 4));
  if (wide) {
    if (rank <= 32) hipLaunchKernelGGL((k_adapter_up<2, 1, 4>), up_grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_adapter_up<2, 2, 4>), up_grid, block, 0, stream, a);
  } else {
    if (rank <= 32) hipLaunchKernelGGL((k_adapter_up<1, 1, 2>), up_grid, block, 0, stream, a);
    else if (rank <= 64) hipLaunchKernelGGL((k_adapter_up<1, 2, 2>), up_grid, block, 0, stream, a);
    else if (rank <= 128) hipLaunchKernelGGL((k_adapter_up<1, 4, 2>), up_grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_adapter_up<1, 8, 2>), up_grid, block, 0, stream, a);
  }
  return m2r_check(hipGetLastError(), "adapters up launch");
}
