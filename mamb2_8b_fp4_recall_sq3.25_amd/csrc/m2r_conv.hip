// Short causal convolution with SiLU over a pool of windows, for gfx950: the
// step before the ragged scan (m2r_full.hip), with the same slots and lengths.
//   o_t = half(silu(bias + sum_{j<4} w_j u_{t-3+j})),
// u before a row's first token being its window's last three inputs; the
// window then holds the row's last four inputs.
//
// A thread takes 8 channels (16 bytes of a token's row) and up to 32 tokens in
// a row, eight at a time with the next eight on their way; the three before
// them stay in registers.  Bound by memory: 4 bytes a channel and token.
// 10,240 channels: 8,192 tokens of one row 76 us, 4.4 TB/s, where a large copy
// has 5.0; nine rows of 62 to 901 tokens, padded to 901, 49 us; one token of 64
// rows 6 us.
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

// x / (1 + exp(-x)) in binary32 with the hardware's exponential and reciprocal,
// for a result that is rounded to binary16 (2^-11).  x log2(e), rounded, is off
// by up to 1.22 |x| 2^-24 as a natural exponent (the constant's own 2^-26.2 with
// it), the other operations by up to 6 times 2^-24: for x >= -21 the result is
// within 2^-19 of the value.  Below, value and result are under 2^-25, half of
// binary16's least, and become zeros (from about -88 on the exponential is
// infinite and the result -0).
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}

// TOKENS: of a thread, STEP of them at a time.
template <int VEC, int TOKENS, int STEP>
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
  const int64_t os = a.n[part];
  uint16_t* out = a.out[part] + (b * a.tokens + t0) * os + at;
  const int64_t end = a.tokens - t0 < TOKENS ? a.tokens - t0 : TOKENS;   // of the outputs
  int64_t done = 0;
  if (t0 < live) {
    const uint16_t* value = a.value + b * a.vs_b + c;
    const int64_t last = live - 1 - t0;      // of this thread's tokens
    V u[STEP + 3], next[STEP];
    auto load = [&](int64_t from) {          // past the end the last token again, not used
#pragma unroll
      for (int i = 0; i < STEP; ++i) next[i] = *(const V*)(value + (t0 + (from + i < last ? from + i : last)) * a.vs_l);
    };
    load(0);
    if (t0 == 0) {
      // this thread alone reads and writes its channels of the row's window
      uint16_t* window = a.window + slot * a.ws_s + c;
#pragma unroll
      for (int j = 0; j < 3; ++j) u[j] = *(const V*)(window + (j + 1) * a.ws_t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t s = live - 4 + j;      // -1 ... -3: the window's last three
        V v = *(const V*)(value + (s > 0 ? s : 0) * a.vs_l);
        if (s == -1) v = u[2];
        if (s == -2) v = u[1];
        if (s == -3) v = u[0];
        *(V*)(window + j * a.ws_t) = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) u[j] = *(const V*)(value + (t0 - 3 + j) * a.vs_l);
    }
    Halves<4> wk[VEC];
    float bk[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      wk[k] = *(const Halves<4>*)(a.weight + 4 * (c + k));
      bk[k] = a.bias ? h2f(a.bias[c + k]) : 0.f;
    }
    const int64_t mine = last + 1 < end ? last + 1 : end;
    for (; done < mine; done += STEP) {
#pragma unroll
      for (int i = 0; i < STEP; ++i) u[3 + i] = next[i];
      if (TOKENS > STEP && done + STEP < mine) load(done + STEP);
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        V o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float s = bk[k];
#pragma unroll
          for (int j = 0; j < 4; ++j) s = __builtin_fmaf(h2f(wk[k].v[j]), h2f(u[i + j].v[k]), s);
          o.v[k] = f2h(a.silu ? silu(s) : s);
        }
        if (done + i < mine) *(V*)(out + (done + i) * os) = o;
      }
#pragma unroll
      for (int j = 0; j < 3; ++j) u[j] = u[STEP + j];
    }
    done = mine;
  }
  for (; done < end; ++done) *(V*)(out + done * os) = V{};
}

template <int VEC, int TOKENS, int STEP>
static int conv_launch(ConvArgs& a, hipStream_t stream) {
  const int64_t cb = (a.C + 256 * VEC - 1) / (256 * VEC), tb = (a.tokens + TOKENS - 1) / TOKENS;
  if (cb * tb > 0x7fffffff / a.batch || !m2r_grid_fits(cb * tb * a.batch, 256))
    return m2r_fail("conv pool: grid limits exceeded");
  a.channel_blocks = (uint32_t)cb;
  a.token_blocks = (uint32_t)tb;
  hipLaunchKernelGGL((k_conv_pool<VEC, TOKENS, STEP>), dim3((unsigned)(cb * tb * a.batch)), dim3(256), 0, stream, a);
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
  if (tokens == 1) return wide ? conv_launch<8, 1, 1>(a, stream) : conv_launch<1, 1, 1>(a, stream);
  if (!wide) return conv_launch<1, 8, 8>(a, stream);
  // 32 tokens a thread once that leaves a workgroup a CU.  us with 8 a thread (11 loads for 8 outputs) / 32, 10,240
  // channels: 8,192 tokens of one row 101 / 76, 1,000 of three 39 / 30, 128 of 16 27 / 24, 200 of four 14 / 16, 500 of
  // one 11 / 15, 77 of one 6 / 13
  const int64_t blocks = (C + 2047) / 2048 * batch * ((tokens + 31) / 32);
  return blocks >= 256 ? conv_launch<8, 32, 8>(a, stream) : conv_launch<8, 8, 8>(a, stream);
}
