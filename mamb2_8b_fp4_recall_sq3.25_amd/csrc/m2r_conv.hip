// Short causal convolution with SiLU over a pool of windows, for gfx950: the
// step before the ragged scan (m2r_full.hip), with the same slots and lengths.
//   o_t = half(silu(bias + sum_{j<4} w_j u_{t-3+j})),
// u before a row's first token being its window's last three inputs; the
// window then holds the row's last four inputs.
//
// A thread takes 8 channels (16 bytes of a token's row) and kTokens tokens in
// a row, so that an input is read once from memory and its three neighbours
// stay in registers.  Bound by memory: 4 bytes a channel and token.
#include "m2r_device.h"
#include "m2r_abi_util.h"

#include <initializer_list>

namespace m2r {

struct ConvArgs {
  uint16_t* window;
  int64_t pool, ws_s, ws_t;
  const uint16_t* value;
  int64_t vs_b, vs_l;
  const uint16_t *weight, *bias;
  const int32_t *slots, *lengths;
  uint16_t* out[3];
  int64_t n[3];
  int64_t C, batch, tokens;
  uint32_t channel_blocks, token_blocks;
  int silu;
};

template <int VEC>
struct alignas(2 * VEC) Halves { uint16_t v[VEC]; };

// x / (1 + exp(-x)) in binary32: the exponential and the reciprocal are the
// hardware's, within 2^-20 of the value, against binary16's 2^-11.
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}

template <int VEC, int TOKENS>
__global__ __launch_bounds__(256) void k_conv_pool(ConvArgs a) {
  typedef Halves<VEC> V;
  uint32_t w = blockIdx.x;
  const uint32_t cb = w % a.channel_blocks;
  w /= a.channel_blocks;
  const int64_t t0 = (int64_t)(w % a.token_blocks) * TOKENS, b = w / a.token_blocks;
  const int64_t c = ((int64_t)cb * 256 + threadIdx.x) * VEC;
  if (c >= a.C) return;
  const int64_t slot = a.slots ? a.slots[b] : b;
  int64_t live = a.lengths ? a.lengths[b] : a.tokens;
  live = slot < 0 || slot >= a.pool || live < 0 ? 0 : (live < a.tokens ? live : a.tokens);
  int part = 0;
  int64_t at = c;
  while (part < 2 && at >= a.n[part]) at -= a.n[part++];
  uint16_t* out = a.out[part] + (b * a.tokens + t0) * a.n[part] + at;
  const int64_t os = a.n[part];

  float y[TOKENS][VEC] = {};
  if (t0 < live) {
    const uint16_t* value = a.value + b * a.vs_b + c;
    V u[TOKENS + 3];
    if (t0 == 0) {
      // this thread alone reads and writes its channels of the row's window
      uint16_t* window = a.window + slot * a.ws_s + c;
#pragma unroll
      for (int j = 0; j < 3; ++j) u[j] = *(const V*)(window + (j + 1) * a.ws_t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t s = live - 4 + j;   // -1 ... -3: the window's last three
        V last = *(const V*)(value + (s > 0 ? s : 0) * a.vs_l);
        if (s == -1) last = u[2];
        if (s == -2) last = u[1];
        if (s == -3) last = u[0];
        *(V*)(window + j * a.ws_t) = last;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) u[j] = *(const V*)(value + (t0 - 3 + j) * a.vs_l);
    }
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {   // past the end the last row's token again, not stored
      const int64_t t = t0 + i < live ? t0 + i : live - 1;
      u[3 + i] = *(const V*)(value + t * a.vs_l);
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const Halves<4> wk = *(const Halves<4>*)(a.weight + 4 * (c + k));
      const float bk = a.bias ? h2f(a.bias[c + k]) : 0.f;
#pragma unroll
      for (int i = 0; i < TOKENS; ++i) {
        float s = bk;
#pragma unroll
        for (int j = 0; j < 4; ++j) s = __builtin_fmaf(h2f(wk.v[j]), h2f(u[i + j].v[k]), s);
        y[i][k] = a.silu ? silu(s) : s;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    if (t0 + i >= a.tokens) break;
    V o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = t0 + i < live ? f2h(y[i][k]) : 0;
    *(V*)(out + i * os) = o;
  }
}

template <int VEC, int TOKENS>
static int conv_launch(ConvArgs& a, hipStream_t stream) {
  const int64_t cb = (a.C + 256 * VEC - 1) / (256 * VEC), tb = (a.tokens + TOKENS - 1) / TOKENS;
  if (cb * tb > 0x7fffffff / a.batch) return m2r_fail("conv pool: grid limits exceeded");
  a.channel_blocks = (uint32_t)cb;
  a.token_blocks = (uint32_t)tb;
  hipLaunchKernelGGL((k_conv_pool<VEC, TOKENS>), dim3((unsigned)(cb * tb * a.batch)), dim3(256), 0, stream, a);
  return m2r_check(hipGetLastError(), "conv pool launch");
}

}  // namespace m2r

using namespace m2r;

extern "C" int m2r_conv_pool(void* window, int64_t pool, int64_t ws_s, int64_t ws_t, const void* value, int64_t vs_b,
                             int64_t vs_l, const void* weight, const void* bias, const int32_t* slots,
                             const int32_t* lengths, void* x, void* bm, void* cm, int64_t n_x, int64_t n_b,
                             int64_t n_c, int64_t batch, int64_t tokens, int width, int silu, hipStream_t stream) {
  if (pool <= 0 || n_x <= 0 || n_b <= 0 || n_c <= 0 || batch <= 0 || tokens <= 0)
    return m2r_fail("conv pool: non-positive shape");
  if (width != 4) return m2r_fail("conv pool: width must be 4");
  const int64_t lim = (int64_t)1 << 24, C = n_x + n_b + n_c;
  if (n_x > lim || n_b > lim || n_c > lim || batch > lim || tokens > lim || pool > lim)
    return m2r_fail("conv pool: size limits");
  for (const void* p : {(const void*)window, value, weight, (const void*)x, (const void*)bm, (const void*)cm})
    if (!p) return m2r_fail("conv pool: null pointer");
  if (!slots && pool < batch) return m2r_fail("conv pool: more batch rows than windows");
  if (ws_t < C || (pool > 1 && ws_s < 3 * ws_t + C)) return m2r_fail("conv pool: windows overlap");
  if (vs_b < 0 || vs_l < 0) return m2r_fail("conv pool: negative strides");
  if ((uintptr_t)weight & 7) return m2r_fail("conv pool: weight must be 8-byte aligned");
  ConvArgs a{(uint16_t*)window, pool, ws_s, ws_t, (const uint16_t*)value, vs_b, vs_l, (const uint16_t*)weight,
             (const uint16_t*)bias, slots, lengths, {(uint16_t*)x, (uint16_t*)bm, (uint16_t*)cm}, {n_x, n_b, n_c}, C,
             batch, tokens, 0, 0, silu};
  const uint64_t bases = (uintptr_t)window | (uintptr_t)value | (uintptr_t)x | (uintptr_t)bm | (uintptr_t)cm;
  const bool wide = !(bases & 15) && !((ws_s | ws_t | vs_b | vs_l | n_x | n_b | n_c) & 7);
  if (tokens == 1) return wide ? conv_launch<8, 1>(a, stream) : conv_launch<1, 1>(a, stream);
  return wide ? conv_launch<8, 8>(a, stream) : conv_launch<1, 8>(a, stream);
}
