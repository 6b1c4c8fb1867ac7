// Token sampling with temperature, top-k, top-p and min-p from one given
// uniform number a row, for gfx950.
//
// Per row, with top = the largest logit and rate = log2(e) / temperature:
//   w_i  = floor(2^31 2^(-(top - l_i) rate)),  a whole number;
// the filters each keep a prefix of the row sorted by (logit descending,
// index ascending): top-k its first k tokens; top-p the shortest prefix that
// holds ceil(top_p W_k) of the weight W_k that top-k left; min-p the tokens
// with w_i >= ceil(min_p 2^31).  The token is the first one, in the order of
// the indices, at which the running sum of the kept weights exceeds
// floor(u W).  Weights are whole numbers so that every sum is exact: the
// result does not depend on how a row is split, nor on the order in which
// atomics arrive.  A token below 2^-31 of the likeliest one is never drawn.
#include "m2r_device.h"
#include "m2r_abi_util.h"

namespace m2r {

enum { LOGITS_F16 = 0, LOGITS_BF16 = 1, LOGITS_F32 = 2 };

struct SampleArgs {
  const void* logits;
  int64_t ls;          // element stride of rows
  const float* u;
  const float *temperature, *top_p, *min_p;   // per row, or null: the scalars
  const int32_t* top_k;
  float temperature_s, top_p_s, min_p_s;
  int32_t top_k_s;
  int64_t* ids;
  float* logprobs;
  int64_t batch, V;
};

// A NaN counts as -inf (never drawn), -0 as +0.
template <int DT>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
  float f;
  if constexpr (DT == LOGITS_F32) f = ((const float*)row)[i];
  else if constexpr (DT == LOGITS_F16) f = h2f(((const uint16_t*)row)[i]);
  else f = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[i] << 16);
  return f != f ? -__builtin_inff() : f + 0.0f;
}

// Order-preserving map of a binary32 value (no NaN, no -0) to 32 bits.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

struct RowFilter {
  float top, rate;
  int64_t k;           // V where top-k is off
  double p;
  uint32_t least;      // min-p: the smallest weight kept (at least 1)
};

__device__ __forceinline__ RowFilter row_filter(const SampleArgs& a, int64_t row) {
  const float t = a.temperature ? a.temperature[row] : a.temperature_s;
  const int64_t k = a.top_k ? a.top_k[row] : a.top_k_s;
  const float p = a.top_p ? a.top_p[row] : a.top_p_s, m = a.min_p ? a.min_p[row] : a.min_p_s;
  const bool greedy = !(t > 0.f);   // the likeliest token, the lowest index of several
  RowFilter f;
  f.top = -__builtin_inff();
  f.rate = (1.0f / (greedy ? 1.0f : t)) * 0x1.715476p+0f;
  f.k = greedy ? 1 : (k > 0 && k < a.V ? k : a.V);
  f.p = p < 1.f ? (double)p : 1.0;
  const double least = m > 0.f ? __builtin_ceil((m < 1.f ? (double)m : 1.0) * 0x1p31) : 1.0;
  f.least = least > 1.0 ? (uint32_t)least : 1u;
  return f;
}

__device__ __forceinline__ uint32_t weight_of(const RowFilter& f, float l) {
  const float away = l == f.top ? 0.0f : (f.top - l) * f.rate;
  return away < 32.0f ? (uint32_t)(__builtin_amdgcn_exp2f(-away) * 0x1p31f) : 0u;
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int by) {
  const uint32_t lo = __shfl_up((uint32_t)v, by), hi = __shfl_up((uint32_t)(v >> 32), by);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {   // inclusive
  const int lane = threadIdx.x & 63;
  for (int by = 1; by < 64; by *= 2) {
    const uint64_t o = shfl_up64(v, by);
    if (lane >= by) v += o;
  }
  return v;
}

constexpr int kRowThreads = 1024;

struct RowShared {
  uint32_t cnt[256];
  uint64_t sum[256];
  uint64_t part[kRowThreads / 64];
  float fpart[kRowThreads / 64];
  uint64_t found[4];   // digit, tokens before it, weight before it
};

// Exclusive prefix sum over the workgroup; `total` receives the sum.
__device__ __forceinline__ uint64_t block_scan64(RowShared& s, uint64_t v, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t inc = wave_scan64(v);
  __syncthreads();
  if (lane == 63) s.part[w] = inc;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
  for (int i = 0; i < kRowThreads / 64; ++i) {
    if (i < w) before += s.part[i];
    total += s.part[i];
  }
  return before + inc - v;
}

struct Cut { uint32_t key; uint64_t count, weight; };   // tokens and weight before the key's first one

// The key at which the sorted row's running count (BY_WEIGHT: weight) reaches
// `target`, digit by digit; tokens of weight 0 do not count.  The target must
// be reached.
template <int DT, bool BY_WEIGHT>
__device__ Cut select_key(RowShared& s, const void* row, int64_t V, const RowFilter& f, uint64_t target) {
  Cut c{0, 0, 0};
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) {
      s.cnt[threadIdx.x] = 0;
      s.sum[threadIdx.x] = 0;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < V; i += kRowThreads) {
      const float l = load_logit<DT>(row, i);
      const uint32_t key = order_key(l), w = weight_of(f, l);
      if (w && (shift == 24 || (key >> (shift + 8)) == (c.key >> (shift + 8)))) {
        atomicAdd(&s.cnt[(key >> shift) & 255], 1u);
        atomicAdd((unsigned long long*)&s.sum[(key >> shift) & 255], (unsigned long long)w);
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {   // lane i: digits 255 - 4 i down to 252 - 4 i
      const int d0 = 255 - 4 * (int)threadIdx.x;
      uint64_t n = 0, w = 0;
      for (int j = 0; j < 4; ++j) {
        n += s.cnt[d0 - j];
        w += s.sum[d0 - j];
      }
      uint64_t nb = c.count + wave_scan64(n) - n, wb = c.weight + wave_scan64(w) - w;
      for (int j = 0; j < 4; ++j) {
        const uint64_t nn = nb + s.cnt[d0 - j], ww = wb + s.sum[d0 - j];
        if (BY_WEIGHT ? wb < target && target <= ww : nb < target && target <= nn) {
          s.found[0] = d0 - j;
          s.found[1] = nb;
          s.found[2] = wb;
        }
        nb = nn;
        wb = ww;
      }
    }
    __syncthreads();
    c.key |= (uint32_t)s.found[0] << shift;
    c.count = s.found[1];
    c.weight = s.found[2];
  }
  return c;
}

// One workgroup per row.
template <int DT>
__global__ __launch_bounds__(kRowThreads) void k_sample_row(SampleArgs a) {
  __shared__ RowShared s;
  const int64_t r = blockIdx.x, V = a.V;
  const int tid = threadIdx.x, lane = tid & 63;
  const void* row = (const char*)a.logits + r * a.ls * (DT == LOGITS_F32 ? 4 : 2);
  RowFilter f = row_filter(a, r);
  float top = -__builtin_inff();
  for (int64_t i = tid; i < V; i += kRowThreads) top = __builtin_fmaxf(top, load_logit<DT>(row, i));
  for (int by = 32; by; by >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, by));
  if (lane == 0) s.fpart[tid >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kRowThreads / 64; ++i) top = __builtin_fmaxf(top, s.fpart[i]);
  if (top == -__builtin_inff()) {   // every token masked
    if (tid == 0) {
      a.ids[r] = -1;
      a.logprobs[r] = -__builtin_inff();
    }
    return;
  }
  f.top = top;

  // the cut: tokens of larger keys, and the first `ties` tokens of its key
  uint32_t cut = 0;
  uint64_t ties = ~0ull;
  uint64_t n = 0, w = 0, positive, all;
  for (int64_t i = tid; i < V; i += kRowThreads) {
    const uint32_t wi = weight_of(f, load_logit<DT>(row, i));
    n += wi != 0;
    w += wi;
  }
  block_scan64(s, n, positive);
  block_scan64(s, w, all);
  if ((uint64_t)f.k < positive) {
    const Cut c = select_key<DT, false>(s, row, V, f, f.k);
    cut = c.key;
    ties = f.k - c.count;
    const uint32_t b = cut ^ ((cut >> 31) ? 0x80000000u : 0xffffffffu);
    all = c.weight + ties * weight_of(f, __builtin_bit_cast(float, b));
  }
  if (f.p < 1.0) {
    const double m = __builtin_ceil(f.p * (double)all);
    const uint64_t mass = m > 1.0 ? (uint64_t)m : 1;
    const Cut c = select_key<DT, true>(s, row, V, f, mass);
    const uint32_t b = c.key ^ ((c.key >> 31) ? 0x80000000u : 0xffffffffu);
    const uint64_t each = weight_of(f, __builtin_bit_cast(float, b)), t = (mass - c.weight + each - 1) / each;
    cut = c.key;      // at or above the top-k cut: mass <= all
    ties = t;
  }

  // the draw: a thread's tokens are neighbours
  const int64_t per = (V + kRowThreads - 1) / kRowThreads, i0 = tid * per, i1 = i0 + per < V ? i0 + per : V;
  uint64_t equal = 0, unused;
  for (int64_t i = i0; i < i1; ++i) equal += order_key(load_logit<DT>(row, i)) == cut;
  const uint64_t rank0 = block_scan64(s, equal, unused);
  uint64_t rank = rank0, kept = 0, total;
  for (int64_t i = i0; i < i1; ++i) {
    const float l = load_logit<DT>(row, i);
    const uint32_t key = order_key(l), wi = weight_of(f, l);
    if ((key > cut || (key == cut && rank < ties)) && wi >= f.least) kept += wi;
    rank += key == cut;
  }
  const uint64_t before = block_scan64(s, kept, total);
  const double at = __builtin_floor((double)a.u[r] * (double)total);
  uint64_t target = at > 0.0 ? (uint64_t)at : 0;
  target = target < total ? target : total - 1;
  if (before <= target && target < before + kept) {
    uint64_t run = before;
    rank = rank0;
    for (int64_t i = i0; i < i1; ++i) {
      const float l = load_logit<DT>(row, i);
      const uint32_t key = order_key(l), wi = weight_of(f, l);
      if ((key > cut || (key == cut && rank < ties)) && wi >= f.least) run += wi;
      rank += key == cut;
      if (run > target) {
        a.ids[r] = i;
        const float away = l == f.top ? 0.0f : (f.top - l) * f.rate;
        a.logprobs[r] = -away * 0x1.62e43p-1f - logf((float)total * 0x1p-31f);
        break;
      }
    }
  }
}

}  // namespace m2r

using namespace m2r;

extern "C" int64_t m2r_sample_workspace(int64_t batch, int64_t V) { return 0; }

extern "C" int m2r_sample(const void* logits, int dtype, int64_t row_stride, const float* uniforms,
                          const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                          const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* ids,
                          float* logprobs, int64_t batch, int64_t V, void* workspace, int64_t workspace_bytes,
                          hipStream_t stream) {
  if (batch <= 0 || V <= 0) return m2r_fail("sample: non-positive shape");
  if (batch > 0x7fffffff || V > 0x7fffffff) return m2r_fail("sample: size limits");
  if (!logits || !uniforms || !ids || !logprobs) return m2r_fail("sample: null pointer");
  if (row_stride < V && batch > 1) return m2r_fail("sample: rows overlap");
  SampleArgs a{logits, row_stride, uniforms, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all,
               top_k_all, ids, logprobs, batch, V};
  const dim3 grid((unsigned)batch), block(kRowThreads);
  if (dtype == LOGITS_F16) hipLaunchKernelGGL(k_sample_row<LOGITS_F16>, grid, block, 0, stream, a);
  else if (dtype == LOGITS_BF16) hipLaunchKernelGGL(k_sample_row<LOGITS_BF16>, grid, block, 0, stream, a);
  else if (dtype == LOGITS_F32) hipLaunchKernelGGL(k_sample_row<LOGITS_F32>, grid, block, 0, stream, a);
  else return m2r_fail("sample: logits must be binary16 (0), bfloat16 (1) or binary32 (2)");
  return m2r_check(hipGetLastError(), "sample launch");
}
