// Selective-state scan with a full-precision (binary32) carry for gfx950:
// linear attention with a decay for each head, as the Mamba-2 mixer runs it
// when no codec holds its carry.  Per head h of batch row b:
//   dt_t = softplus(dt[b, t, h] + dt_bias[h]),  a_t = exp(A[h] dt_t)
//   S_t  = a_t S_{t-1} + dt_t x_t (x) B_t            (S: [P, 128])
//   y_t  = half(S_t C_t + D[h] x_t)
// Operands and readouts are binary16 as the model holds them; dt, decays,
// carries and sums are binary32, and a readout is rounded once.  A few tokens
// are stepped one by one (k_full_rows, here); more go through the matrix cores
// in chunks (m2r_full_chunks.hip).
#include "m2r_full.h"
#include "m2r_abi_util.h"

#include <initializer_list>

namespace m2r {

typedef uint16_t h16x4 __attribute__((ext_vector_type(4)));

// Token by token.  Half a wave holds one row of the carry (lane n holds
// coordinates 4n .. 4n + 3, a 16-byte access), a wave 2 R rows, so that R
// loads of 1 KiB are in flight; the readout is a butterfly over 32 lanes.
// One token is bound by memory: it reads and writes 1 KiB of carry a row for
// 640 operations.  At 128 heads of 64, 61 of 64 batch rows at work, 514 MB: 91
// to 94 us among calls in one graph, 5.5 TB/s, where a copy of 2 GiB reaches
// 4.9; a graph of one call 99 (R = 2: 108 us, fewer loads in flight; R = 8: 104,
// fewer waves).  Batch 1, 8.4 MB: 4.3 us, a launch and one way to memory and
// back; a graph of one call 5.3 (R = 2: 5.4, R = 8: 6.1).
template <int R>
__global__ __launch_bounds__(256) void k_full_rows(FullArgs a) {
  const int lane = threadIdx.x & 63, half = lane >> 5, q = lane & 31;
  const int64_t blocks = (a.P + 2 * R - 1) / (2 * R);
  int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= a.batch * a.H * blocks) return;
  const int64_t p0 = (w % blocks) * 2 * R;
  w /= blocks;
  const int64_t h = w % a.H, b = w / a.H;
  const int64_t g = h / (a.H / a.G);
  const FullRow fr = full_row(a, b);
  const int64_t slot = fr.slot, len = fr.len;
  // the lane that stores row 2 q + half of the wave's rows
  const bool writer = q < R && p0 + 2 * q + half < a.P;
  uint16_t* y = a.y + (b * a.L * a.H + h) * a.P + p0 + 2 * q + half;
  if (len > 0) {
    float* srow = a.state + ((slot * a.H + h) * a.P + p0 + half) * 128 + 4 * q;
    f32x4 s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = p0 + 2 * r + half < a.P ? *(const f32x4*)(srow + 256 * r) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float av = a.A[h];
    const FullParam skip = full_param(a.D, a.d_f32, h), bias = full_param(a.dt_bias, a.db_f32, h);
    const uint16_t* xp = a.x + b * a.xs_b + h * a.P + p0 + half;
    const uint16_t* dp = a.dt + b * a.ds_b + h;
    const uint16_t* bp = a.Bm + b * a.bs_b + g * 128 + 4 * q;
    const uint16_t* cp = a.Cm + b * a.cs_b + g * 128 + 4 * q;
    for (int64_t t = 0; t < len; ++t) {
      const float dt = full_dt(h2f(dp[t * a.ds_l]) + bias.value());
      const float decay = expf(av * dt);
      const uint16_t *bt = bp + t * a.bs_l, *ct = cp + t * a.cs_l;
      float bv[4], cv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bv[j] = h2f(bt[j]);
        cv[j] = h2f(ct[j]);
      }
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float xv = p0 + 2 * r + half < a.P ? h2f(xp[t * a.xs_l + 2 * r]) : 0.f;
        const float in = xv * dt;
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[r][j] = __builtin_fmaf(s[r][j], decay, in * bv[j]);
          acc = __builtin_fmaf(s[r][j], cv[j], acc);
        }
        acc = butterfly_add<4>(butterfly_add<3>(butterfly_add<2>(butterfly_add<1>(butterfly_add<0>(acc)))));
        if (q == r) mine = __builtin_fmaf(xv, skip.value(), acc);
      }
      if (writer) y[t * a.H * a.P] = f2h(mine);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (p0 + 2 * r + half < a.P) *(f32x4*)(srow + 256 * r) = s[r];
  }
  if (writer)
    for (int64_t t = len; t < a.L; ++t) y[t * a.H * a.P] = 0;
}

}  // namespace m2r

using namespace m2r;

// Whether a call of L tokens takes the chunked kernel, whose time hardly
// depends on L up to 64, or steps token by token.  The step's time is its
// carries' plus a chain per token; few rows leave the chain bare, so the
// chunked kernel's fixed cost is made up later.  us per call, step / chunked,
// at 128 heads of 64: batch 1 12 tokens 15.5 / 18.8, 16 tokens 19.0 / 18.4;
// batch 4 8 tokens 18.5 / 20.6, 12 tokens 24.0 / 20.2; batch 16 4 tokens
// 35.7 / 43.7, 6 tokens 44.6 / 44.2; batch 64 4 tokens 134 / 162, 6 tokens
// 168 / 157, 64 tokens 1,253 / 183.
static bool full_chunked(int64_t batch, int64_t L, int64_t H, int64_t P) {
  const int64_t rows = batch * H * P;
  return L >= (rows <= 16384 ? 16 : (rows <= 65536 ? 10 : 6));
}

extern "C" int64_t m2r_full_scan_workspace(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G) {
  if (batch <= 0 || H <= 0 || P <= 0 || G <= 0 || H % G || batch > 65535 || !full_chunked(batch, L, H, P)) return 0;
  return full_chunks_workspace(batch, L, H, P, G);
}

extern "C" int m2r_full_scan(const void* x, int64_t xs_b, int64_t xs_l, const void* dt, int64_t ds_b, int64_t ds_l,
                             const float* A, const void* B, int64_t bs_b, int64_t bs_l, const void* C, int64_t cs_b,
                             int64_t cs_l, const void* D, int d_is_f32, const void* dt_bias, int db_is_f32,
                             float* state, int64_t pool, const int32_t* slots, const int32_t* lengths, void* y,
                             int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G, void* workspace,
                             int64_t workspace_bytes, hipStream_t stream) {
  if (batch <= 0 || L <= 0 || H <= 0 || P <= 0 || G <= 0 || pool <= 0 || H % G) return m2r_fail("full scan: bad geometry");
  const int64_t lim = (int64_t)1 << 24;
  if (batch > lim || L > lim || H > lim || P > lim || pool > ((int64_t)1 << 31) ||
      (__int128)batch * L * H * P >= (__int128)1 << 60 || (__int128)pool * H * P >= (__int128)1 << 50)
    return m2r_fail("full scan: size limits");
  if (!slots && batch > pool) return m2r_fail("full scan: more batch rows than carries");
  for (const void* p : {x, dt, (const void*)A, B, C, D, dt_bias, (const void*)state, (const void*)y})
    if (!p) return m2r_fail("full scan: null pointer");
  if ((uintptr_t)state & 15) return m2r_fail("full scan: the carry must be 16-byte aligned");
  FullArgs a{(const uint16_t*)x, (const uint16_t*)dt, xs_b, xs_l, ds_b, ds_l, A, (const uint16_t*)B,
             (const uint16_t*)C, bs_b, bs_l, cs_b, cs_l, D, dt_bias, d_is_f32, db_is_f32, state, pool, slots, lengths,
             (uint16_t*)y, batch, L, H, P, G};
  // (a grid's second axis holds the batch rows)
  if (batch <= 65535 && full_chunked(batch, L, H, P)) {
    const int64_t need = full_chunks_workspace(batch, L, H, P, G);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
      return m2r_fail("full scan: workspace too small or not 16-byte aligned");
    return m2r_check(launch_full_chunks(a, workspace, stream), "full scan launch");
  }
  constexpr int R = 4;
  const __int128 waves = (__int128)batch * H * ((P + 2 * R - 1) / (2 * R));
  if ((waves + 3) / 4 > 0x7fffffff) return m2r_fail("full scan: grid limits exceeded");
  hipLaunchKernelGGL(k_full_rows<R>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, a);
  return m2r_check(hipGetLastError(), "full scan launch");
}
