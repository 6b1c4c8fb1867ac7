// Penalties for repeated tokens, biases and grammar masks on logits, for
// gfx950, before a token is drawn from them (m2r_sample.hip).  For a row's
// token v, c times among its generated tokens:
//   l <- l / r (l > 0) or l r (else)   where v is in the prompt or c > 0
//   l <- l - (f c + p)                 where c > 0
//   l <- l + bias[v]                   the last entry of the row's list that names v
//   l <- -inf                          where the row's mask does not allow v
// in binary32, rounded once to the logits' type; a logit that none of this
// touches keeps its bits.
//
// A workgroup takes a slice of a row's tokens.  It counts the row's ids that
// lie in its slice in a table in LDS (whole numbers: the order does not
// matter), then passes over its logits once, which were on their way meanwhile;
// no counts are kept in memory.  Bound by memory: each logit read and written
// once.  64 rows of 256,000 in binary32 with lists, biases and masks 32 us, 4.2
// TB/s; one row of binary16 4.3 us.  With long lists every slice reads all ids
// of its row (8 rows with up to 104,000 ids: 17 us, a thread's 100 ids and their
// counting; plain stores of the prompt's flags in place of atomics, twice as many
// loads in flight and other slices changed nothing).
#include "m2r_device.h"
#include "m2r_abi_util.h"

namespace m2r {

struct IdList {
  const void* ids;       // int32 or int64 rows, or null
  int64_t stride, n;
  const int32_t* lengths;
  int wide;              // 1: int64
};
struct alignas(16) Word4 { uint32_t w[4]; };
struct RowValue {
  const float* row;      // a value for each row, or null
  float all;
};
struct AdjustArgs {
  const void* logits;
  int64_t ls;
  void* out;
  int64_t os;
  IdList prompt, tokens;
  RowValue repetition, presence, frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_ids_stride, bias_values_stride, biases;
  const uint32_t* allowed;
  int64_t allowed_stride, masks;
  const int32_t* allowed_rows;
  int64_t V;
  uint32_t slices;
  int in_place;
};

constexpr uint32_t kInPrompt = 0x80000000u;   // of a table's word; the rest counts the generated tokens

template <int DTYPE> struct LogitType { typedef uint16_t T; };
template <> struct LogitType<2> { typedef float T; };
template <int DTYPE>
__device__ __forceinline__ float logit_value(typename LogitType<DTYPE>::T v) {
  if constexpr (DTYPE == 0) return h2f(v);
  else if constexpr (DTYPE == 1) return __builtin_bit_cast(float, (uint32_t)v << 16);
  else return v;
}
template <int DTYPE>
__device__ __forceinline__ typename LogitType<DTYPE>::T logit_rounded(float v) {
  if constexpr (DTYPE == 0) return f2h(v);
  else if constexpr (DTYPE == 1) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40);   // NaN stays one
    return (uint16_t)((u + 0x7fffu + (u >> 16 & 1)) >> 16);
  } else return v;
}

__device__ __forceinline__ float row_value(const RowValue& v, int64_t row) { return v.row ? v.row[row] : v.all; }

// Calls f(token of the slice) for each id of the row's list in [v0, v0 + size).
// Sixteen bytes of ids a thread, kLoads such loads at a time.
template <int THREADS, int kLoads, typename F>
__device__ __forceinline__ void for_ids(const IdList& l, int64_t row, int64_t v0, int size, F f) {
  if (!l.ids) return;
  int64_t n = l.lengths ? l.lengths[row] : l.n;
  n = n < l.n ? n : l.n;
  const uint32_t from = (uint32_t)v0;
  if (l.wide) {
    const int64_t* p = (const int64_t*)l.ids + row * l.stride;
    for (int64_t i0 = 0; i0 < n; i0 += THREADS * 2 * kLoads) {
      uint64_t id[kLoads][2];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (i0 + j * THREADS * 2 >= n) break;
        const int64_t i = i0 + (j * THREADS + threadIdx.x) * 2;
        if (i + 2 <= n) __builtin_memcpy(id[j], p + i, 16);
        else {
          id[j][0] = i < n ? (uint64_t)p[i] : ~0ull;
          id[j][1] = ~0ull;
        }
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (i0 + j * THREADS * 2 >= n) break;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t at = (uint32_t)id[j][k] - from;
          if (at < (uint32_t)size && !(id[j][k] >> 32)) f((int)at);
        }
      }
    }
  } else {
    const uint32_t* p = (const uint32_t*)l.ids + row * l.stride;
    for (int64_t i0 = 0; i0 < n; i0 += THREADS * 4 * kLoads) {
      uint32_t id[kLoads][4];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (i0 + j * THREADS * 4 >= n) break;
        const int64_t i = i0 + (j * THREADS + threadIdx.x) * 4;
        if (i + 4 <= n) __builtin_memcpy(id[j], p + i, 16);
        else
#pragma unroll
          for (int k = 0; k < 4; ++k) id[j][k] = i + k < n ? p[i + k] : ~0u;
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (i0 + j * THREADS * 4 >= n) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t at = id[j][k] - from;   // (a negative id is above every token)
          if (at < (uint32_t)size) f((int)at);
        }
      }
    }
  }
}

template <int DTYPE, int THREADS, int SLICE, int LOADS>
__global__ __launch_bounds__(THREADS) void k_adjust(AdjustArgs a) {
  typedef typename LogitType<DTYPE>::T T;
  constexpr int VEC = 16 / sizeof(T), ROUNDS = (SLICE + THREADS * VEC - 1) / (THREADS * VEC);
  extern __shared__ __attribute__((aligned(16))) uint32_t table[];   // [SLICE], and [SLICE] places in the list of biases
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.slices, v0 = (int64_t)(blockIdx.x % a.slices) * SLICE;
  const int size = (int)(a.V - v0 < SLICE ? a.V - v0 : SLICE);
  const T* src = (const T*)a.logits + row * a.ls + v0;
  T* dst = (T*)a.out + row * a.os + v0;
  // what the pass over the logits needs is on its way while the ids are counted
  const float repetition = row_value(a.repetition, row), presence = row_value(a.presence, row),
              frequency = row_value(a.frequency, row);
  const uint32_t* allowed = nullptr;
  if (a.allowed) {
    const int64_t m = a.allowed_rows ? a.allowed_rows[row] : row;
    if (m >= 0 && m < a.masks) allowed = a.allowed + m * a.allowed_stride + (v0 >> 5);
  }
  T l[ROUNDS][VEC];
  uint32_t free[ROUNDS];
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const int i = (u * THREADS + tid) * VEC;
    free[u] = allowed && i < size ? allowed[i >> 5] >> (i & 31) : 0xffffffffu;
    if (i + VEC <= size) {
      if (!a.in_place) __builtin_memcpy(l[u], src + i, 16);
    } else
#pragma unroll
      for (int k = 0; k < VEC; ++k) l[u][k] = i + k < size ? src[i + k] : T(0);
  }
  const bool counted = a.prompt.ids || a.tokens.ids, biased = a.bias_ids != nullptr;
  uint32_t* place = table + (counted ? SLICE : 0);
  if (counted || biased) {
    for (int i = 4 * tid; i < SLICE * (counted + biased); i += 4 * THREADS) *(Word4*)(table + i) = Word4{};
    __syncthreads();
    for_ids<THREADS, LOADS>(a.prompt, row, v0, size, [&](int at) { atomicOr(&table[at], kInPrompt); });
    for_ids<THREADS, LOADS>(a.tokens, row, v0, size, [&](int at) { atomicAdd(&table[at], 1u); });
    if (biased)
      for (int64_t i = tid; i < a.biases; i += THREADS) {
        const uint64_t at = (uint64_t)((int64_t)a.bias_ids[row * a.bias_ids_stride + i] - v0);
        if (at < (uint64_t)size) atomicMax(&place[at], (uint32_t)i + 1u);   // the list's last entry for a token
      }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const int i = (u * THREADS + tid) * VEC;
    if (i >= size) continue;
    uint32_t word[VEC], entry[VEC], touched = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      word[k] = counted ? table[i + k] : 0;
      entry[k] = biased ? place[i + k] : 0;
      touched |= word[k] | entry[k];
    }
    const bool all_free = (free[u] & ((1u << VEC) - 1)) == (1u << VEC) - 1, whole = i + VEC <= size;
    if (a.in_place) {
      if (all_free && !touched) continue;
      if (whole) __builtin_memcpy(l[u], src + i, 16);
    }
    if (touched) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        if (!(word[k] | entry[k])) continue;
        float v = logit_value<DTYPE>(l[u][k]);
        if (word[k]) {
          v = v > 0.f ? v / repetition : v * repetition;
          const uint32_t c = word[k] & ~kInPrompt;
          if (c) v = v - (frequency * (float)c + presence);
        }
        if (entry[k]) v = v + a.bias_values[row * a.bias_values_stride + entry[k] - 1];
        l[u][k] = logit_rounded<DTYPE>(v);
      }
    }
    if (!all_free) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (!(free[u] >> k & 1)) l[u][k] = logit_rounded<DTYPE>(-__builtin_inff());
    }
    if (whole) __builtin_memcpy(dst + i, l[u], 16);
    else
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (i + k < size) dst[i + k] = l[u][k];
  }
}

template <int DTYPE, int THREADS, int SLICE, int LOADS>
static int adjust_launch(AdjustArgs& a, int64_t batch, hipStream_t stream) {
  const int64_t slices = (a.V + SLICE - 1) / SLICE;
  if (!m2r_grid_fits(slices * batch, THREADS)) return m2r_fail("adjust: grid limits exceeded");
  a.slices = (uint32_t)slices;
  const size_t lds = 4 * (size_t)SLICE * ((a.prompt.ids || a.tokens.ids) + (a.bias_ids != nullptr));
  static std::atomic<uint64_t> allowed{0};
  if (int rc = m2r_allow_lds((const void*)k_adjust<DTYPE, THREADS, SLICE, LOADS>, 8 * SLICE, allowed)) return rc;
  hipLaunchKernelGGL((k_adjust<DTYPE, THREADS, SLICE, LOADS>), dim3((unsigned)(slices * batch)), dim3(THREADS), lds, stream,
                     a);
  return m2r_check(hipGetLastError(), "adjust launch");
}
template <int DTYPE>
static int adjust_dtype(AdjustArgs& a, int64_t batch, hipStream_t stream) {
  // Threads and slice by the lists' length and the number of workgroups.  us on binary32, 256 x 1,024 /
  // 512 x 4,096 / 1,024 x 4,096 / 1,024 x 16,384:
  //   1 row of 256,000, 1,000 ids     3.7 / 4.5 / 4.1 / 6.4      64 such rows                31 / 28 / 45 / 31
  //   1 row, 50,000 ids                19 / 13 / 8.8 / 12        64 rows, 16,000 ids        100 / 47 / 73 / 46
  //   16 rows of 256,000, 8,000 ids    19 / 12 / 17 / 12         64 rows, 50,000 ids        288 / 104 / 137 / 67
  const int64_t ids = a.prompt.n + a.tokens.n;
  if (ids >= 8192) {
    if (batch * ((a.V + 16383) / 16384) >= 128) return adjust_launch<DTYPE, 1024, 16384, 4>(a, batch, stream);
    return adjust_launch<DTYPE, 1024, 4096, 4>(a, batch, stream);
  }
  if (ids >= 4096 || batch * ((a.V + 4095) / 4096) >= 256) return adjust_launch<DTYPE, 512, 4096, 2>(a, batch, stream);
  return adjust_launch<DTYPE, 256, 1024, 2>(a, batch, stream);
}

}  // namespace m2r

using namespace m2r;

extern "C" int m2r_adjust_logits(const void* logits, int dtype, int64_t row_stride, void* out, int64_t out_stride,
                                 const void* prompt, int prompt_is_i64, int64_t prompt_stride, int64_t prompt_n,
                                 const int32_t* prompt_lengths, const void* tokens, int tokens_are_i64,
                                 int64_t tokens_stride, int64_t tokens_n, const int32_t* lengths,
                                 const float* repetition, float repetition_all, const float* presence,
                                 float presence_all, const float* frequency, float frequency_all,
                                 const int32_t* bias_ids, int64_t bias_ids_stride, const float* bias_values,
                                 int64_t bias_values_stride, int64_t biases, const uint32_t* allowed,
                                 int64_t allowed_stride, int64_t masks, const int32_t* allowed_rows, int64_t batch,
                                 int64_t V, hipStream_t stream) {
  if (batch <= 0 || V <= 0) return m2r_fail("adjust: non-positive shape");
  if (batch > 0x7fffffff || V > 0x7ffffffe) return m2r_fail("adjust: size limits");
  if (dtype < 0 || dtype > 2) return m2r_fail("adjust: logits must be binary16, bfloat16 or binary32");
  if (!logits || !out) return m2r_fail("adjust: null pointer");
  if (row_stride < V || out_stride < V) return m2r_fail("adjust: rows overlap");
  const int64_t lim = (int64_t)1 << 30;
  if (prompt_n < 0 || tokens_n < 0 || biases < 0 || prompt_n > lim || tokens_n > lim || biases > lim)
    return m2r_fail("adjust: list limits");
  if ((prompt_n && !prompt) || (tokens_n && !tokens) || (biases && (!bias_ids || !bias_values)))
    return m2r_fail("adjust: null pointer");
  if (prompt_stride < 0 || tokens_stride < 0 || bias_ids_stride < 0 || bias_values_stride < 0 || allowed_stride < 0)
    return m2r_fail("adjust: negative strides");
  if (allowed && masks <= 0) return m2r_fail("adjust: no masks");
  if (allowed && !allowed_rows && masks < batch) return m2r_fail("adjust: more batch rows than masks");
  AdjustArgs a{logits, row_stride, out, out_stride,
               {prompt_n ? prompt : nullptr, prompt_stride, prompt_n, prompt_lengths, prompt_is_i64},
               {tokens_n ? tokens : nullptr, tokens_stride, tokens_n, lengths, tokens_are_i64},
               {repetition, repetition_all}, {presence, presence_all}, {frequency, frequency_all},
               biases ? bias_ids : nullptr, bias_values, bias_ids_stride, bias_values_stride, biases,
               allowed, allowed_stride, masks, allowed_rows, V, 0, logits == out && row_stride == out_stride};
  if (dtype == 0) return adjust_dtype<0>(a, batch, stream);
  if (dtype == 1) return adjust_dtype<1>(a, batch, stream);
  return adjust_dtype<2>(a, batch, stream);
}
