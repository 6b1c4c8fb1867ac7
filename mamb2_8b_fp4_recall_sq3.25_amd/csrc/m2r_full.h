// Arguments and shared arithmetic of the scan with a full-precision
// (binary32) carry: m2r_full.hip, m2r_full_chunks.hip.
#pragma once
#include "m2r_device.h"
#include "m2r_tile.h"

namespace m2r {

struct FullArgs {
  const uint16_t *x, *dt;
  int64_t xs_b, xs_l, ds_b, ds_l;      // element strides of batch rows and tokens
  const float* A;
  const uint16_t *Bm, *Cm;
  int64_t bs_b, bs_l, cs_b, cs_l;
  const void *D, *dt_bias;
  int d_f32, db_f32;
  float* state;
  int64_t pool;
  const int32_t *slots, *lengths;      // null: row b's carry is b, every row has L tokens
  uint16_t* y;
  int64_t batch, L, H, P, G;
};

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, with
// log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3, by its series to s^15 (the
// rest is below 2^-26 of it).  e keeps the part of v log2(e) that the product
// rounds away, so that small steps have the relative precision of large ones
// (log(exp(v) + 1) in binary32 loses it below v = -8).  NaN and infinities
// come through.
__device__ __forceinline__ float full_dt(float v) {
  constexpr float kLog2e = 0x1.715476p+0f, kLog2eLow = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;
  const float m = -__builtin_fabsf(v), t = m * kLog2e;
  float e = __builtin_amdgcn_exp2f(t);
  const float rest = __builtin_fmaf(m, kLog2eLow, __builtin_fmaf(m, kLog2e, -t));
  e = t > -150.f ? __builtin_fmaf(e, rest * kLn2, e) : 0.f;   // (an infinite m has no rest)
  const float d = 2.0f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  const float s = e * r, q = s * s;
  float p = 1.0f / 15.0f;
  p = __builtin_fmaf(p, q, 1.0f / 13.0f);
  p = __builtin_fmaf(p, q, 1.0f / 11.0f);
  p = __builtin_fmaf(p, q, 1.0f / 9.0f);
  p = __builtin_fmaf(p, q, 1.0f / 7.0f);
  p = __builtin_fmaf(p, q, 1.0f / 5.0f);
  p = __builtin_fmaf(p, q, 1.0f / 3.0f);
  const float l = __builtin_fmaf(s * q, p, s);
  const float y = (v > 0.f ? v : 0.f) + (l + l);
  return v != v ? v : y;
}

// The carry of batch row b, or -1 for an idle row, and its token count (0 for
// an idle row).  Both loads are issued at once, whether they are needed or not.
struct FullRow { int64_t slot, len; };
__device__ __forceinline__ FullRow full_row(const FullArgs& a, int64_t b) {
  const int32_t* any = (const int32_t*)a.A;   // readable, for what is not there
  const int32_t sv = *(a.slots ? a.slots + b : any), lv = *(a.lengths ? a.lengths + b : any);
  const int64_t s = a.slots ? sv : b, n = a.lengths ? lv : a.L;
  FullRow r{s >= 0 && s < a.pool ? s : -1, n < 0 ? 0 : (n < a.L ? n : a.L)};
  if (r.slot < 0) r.len = 0;
  return r;
}

// Element h of a binary16 or binary32 parameter: loaded without a branch, so
// that other loads are issued before it is waited for.
struct FullParam {
  uint16_t low, high;
  int f32;
  __device__ __forceinline__ float value() const {
    return f32 ? __builtin_bit_cast(float, ((uint32_t)high << 16) | low) : h2f(low);
  }
};
__device__ __forceinline__ FullParam full_param(const void* p, int f32, int64_t h) {
  const uint16_t* at = (const uint16_t*)p + (f32 ? 2 * h : h);
  return FullParam{at[0], at[f32 ? 1 : 0], f32};
}

// Many tokens in chunks, on the matrix cores (m2r_full_chunks.hip).
int64_t full_chunks_workspace(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G);
hipError_t launch_full_chunks(const FullArgs& a, void* workspace, hipStream_t stream);

}  // namespace m2r
