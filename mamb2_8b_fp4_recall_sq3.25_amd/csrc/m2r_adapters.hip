// Low-rank adapters of many requests beside a shared projection, for gfx950:
//   out[m] = half(base[m] + scale[a] up[a] (down[a] x[m])),  a = ids[m],
// and out[m] = base[m] where ids[m] names no adapter (negative, or not below
// the number of adapters).  x [M, K], base and out [M, N] binary16 rows,
// down [n, r, K], up [n, N, r] binary16, scale [n] binary32.  The hidden
// values scale[a] (down[a] x[m]) pass between the two kernels in binary32.
#include "m2r_device.h"
#include "m2r_abi_util.h"
#include "m2r_tile.h"

#include <initializer_list>

namespace m2r {

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
  float* hidden;   // [M, r]
  int64_t M, K, N, n;
  int r;
};

// One wave per hidden value.
__global__ __launch_bounds__(256) void k_adapter_down(AdapterArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= a.M * a.r) return;
  const int64_t m = w / a.r, j = w % a.r;
  const int64_t id = a.ids[m];
  if (id < 0 || id >= a.n) return;
  const uint16_t *xr = a.x + m * a.xs, *d = a.down + (id * a.r + j) * a.K;
  float acc = 0.f;
  for (int64_t k = lane; k < a.K; k += 64) acc = __builtin_fmaf(h2f(xr[k]), h2f(d[k]), acc);
  acc = wave_sum(acc);
  if (lane == 0) a.hidden[w] = acc * a.scale[id];
}

// One thread per output.
__global__ __launch_bounds__(256) void k_adapter_up(AdapterArgs a) {
  const int64_t m = blockIdx.y, c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.N) return;
  const int64_t id = a.ids[m];
  uint16_t v = a.base[m * a.bs + c];
  if (id >= 0 && id < a.n) {
    const float* hid = a.hidden + m * a.r;
    const uint16_t* u = a.up + (id * a.N + c) * a.r;
    float acc = 0.f;
    for (int j = 0; j < a.r; ++j) acc = __builtin_fmaf(hid[j], h2f(u[j]), acc);
    v = f2h(h2f(v) + acc);
  }
  a.out[m * a.os + c] = v;
}

}  // namespace m2r

using namespace m2r;

extern "C" int64_t m2r_adapters_workspace(int64_t M, int64_t K, int64_t N, int64_t r) { return 4 * M * r; }

extern "C" int m2r_adapters_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride,
                                const void* down, const void* up, const float* scale, const int32_t* ids, void* out,
                                int64_t out_stride, int64_t M, int64_t K, int64_t N, int64_t adapters, int64_t rank,
                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (M <= 0 || K <= 0 || N <= 0 || adapters <= 0 || rank <= 0) return m2r_fail("adapters: non-positive shape");
  const int64_t lim = (int64_t)1 << 24;
  if (M > lim || K > lim || N > lim || adapters > lim || rank > 256) return m2r_fail("adapters: size limits");
  for (const void* p : {x, base, down, up, (const void*)scale, (const void*)ids, (const void*)out, (const void*)workspace})
    if (!p) return m2r_fail("adapters: null pointer");
  if (x_stride < K || base_stride < N || out_stride < N) return m2r_fail("adapters: rows overlap");
  if ((uintptr_t)workspace & 15 || workspace_bytes < m2r_adapters_workspace(M, K, N, rank))
    return m2r_fail("adapters: workspace too small or not 16-byte aligned");
  AdapterArgs a{(const uint16_t*)x, x_stride, (const uint16_t*)base, base_stride, (const uint16_t*)down,
                (const uint16_t*)up, scale, ids, (uint16_t*)out, out_stride, (float*)workspace, M, K, N, adapters,
                (int)rank};
  if (M > 65535) return m2r_fail("adapters: grid limits exceeded");
  hipLaunchKernelGGL(k_adapter_down, dim3((unsigned)((M * rank + 3) / 4)), dim3(256), 0, stream, a);
  int rc = m2r_check(hipGetLastError(), "adapters down launch");
  if (rc) return rc;
  hipLaunchKernelGGL(k_adapter_up, dim3((unsigned)((N + 255) / 256), (unsigned)M), dim3(256), 0, stream, a);
  return m2r_check(hipGetLastError(), "adapters up launch");
}
