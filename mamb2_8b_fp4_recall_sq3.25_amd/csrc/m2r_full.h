// Arguments and shared arithmetic of the scan with a full-precision
// (binary32) carry: m2r_full.hip.
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

// softplus(v) = log(1 + exp(v)), v itself above 20 (where they agree to
// binary32).  log1p keeps the relative precision of small steps, which
// log(exp(v) + 1) in binary32 loses below v = -8.
__device__ __forceinline__ float full_dt(float v) { return v <= 20.0f ? log1pf(expf(v)) : v; }

// The carry of batch row b, or -1 for an idle row; and its token count.
__device__ __forceinline__ int64_t full_slot(const FullArgs& a, int64_t b) {
  const int64_t s = a.slots ? (int64_t)a.slots[b] : b;
  return s >= 0 && s < a.pool ? s : -1;
}
__device__ __forceinline__ int64_t full_length(const FullArgs& a, int64_t b) {
  if (!a.lengths) return a.L;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : (n < a.L ? n : a.L);
}

// Many tokens in chunks, on the matrix cores (m2r_full_chunks.hip).
int64_t full_chunks_workspace(int64_t batch, int64_t L, int64_t H, int64_t P, int64_t G);
hipError_t launch_full_chunks(const FullArgs& a, void* workspace, hipStream_t stream);

}  // namespace m2r
