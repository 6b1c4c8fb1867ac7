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
// Logits of any type are compared as binary32; sums are 64-bit.
//
// Each logit has to be read once; here it is read two or three times, mostly
// from the caches, since a weight needs the row's largest logit and a cut the
// row's whole weight.  64 rows of 256,000 binary32 logits (65 MB, 13 us for a
// copy), with filters of all kinds: 63 us, the launches 12, 19 and 32.  The
// first two read at 5.3 and 3.4 TB/s; the last ends with its heaviest row (19
// us to gather thousands of listed tokens, then 11 in one workgroup to order
// them and draw).  One row of binary16, filtered: 22 us, three launches of a
// few dependent steps; 24 rows of 50,003 without filters: 11 us.  Logits that
// are all close (normal, deviation 0.02 to 1; top-p 0.9): 64 rows 64 to 70 us,
// where bins of a fixed 1/16 left lists that did not fit (1,350 us).  All
// logits equal, cut by a workgroup a row: one row 143 to 210 us, 64 rows 360 to
// 470 (7,000 with a counter's atomics from every lane).
#include "m2r_device.h"
#include "m2r_abi_util.h"

#include <cstddef>

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

// A NaN counts as -inf (never drawn): the maximum of it and -inf.
__device__ __forceinline__ float no_nan(float f) { return __builtin_fmaxf(f, -__builtin_inff()); }
template <int DT>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
  float f;
  if constexpr (DT == LOGITS_F32) f = ((const float*)row)[i];
  else if constexpr (DT == LOGITS_F16) f = h2f(((const uint16_t*)row)[i]);
  else f = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[i] << 16);
  return no_nan(f);
}

// Order-preserving map of a binary32 value (no NaN; -0 as +0) to 32 bits.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

struct RowFilter {
  float top, rate;
  float fine;          // bins a power of two of weight
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
  f.fine = 0.f;
  // (2^126 stands for whatever lies above, infinity too: at a rate of 0 a masked
  // token, and what is read past the row's end, would weigh as much as the likeliest)
  f.rate = (1.0f / (greedy ? 1.0f : __builtin_fminf(t, 0x1p126f))) * 0x1.715476p+0f;
  f.k = greedy ? 1 : (k > 0 && k < a.V ? k : a.V);
  f.p = p < 1.f ? (double)p : 1.0;
  const double least = m > 0.f ? __builtin_ceil((m < 1.f ? (double)m : 1.0) * 0x1p31) : 1.0;
  f.least = least > 1.0 ? (uint32_t)least : 1u;
  return f;
}

// A token's distance from the largest logit as a power of two.  The maximum
// with 0 answers 0 where the product is 0 * inf or inf - inf, the largest
// logit's own distance.
__device__ __forceinline__ float away_of(const RowFilter& f, float l) {
  return __builtin_fmaxf((f.top - l) * f.rate, 0.0f);
}
// floor(2^31 2^-away); 0 from 32 on by itself.
__device__ __forceinline__ uint32_t weight_at(float away) {
  return (uint32_t)(__builtin_amdgcn_exp2f(-away) * 0x1p31f);
}
__device__ __forceinline__ uint32_t weight_of(const RowFilter& f, float l) { return weight_at(away_of(f, l)); }

__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// ---------------------------------------------------------------------------
// Three launches.  A row is cut into at most kMaxSplits pieces of whole
// 2,048-token blocks, one workgroup each; the kept weight is counted by units
// of at most kUnits a row, a block each but in the longest rows, so that the
// draw reads one of them.
//   k_sample_top:    the largest logit of each piece, and how far below it the
//                    others reach;
//   k_sample_bins:   the row's weight and token counts by 512 bins of the
//                    logit over that range, so that even logits that are all
//                    close leave few in one; the last workgroup of a row then
//                    finds the bins in which top-k and top-p end.  Without
//                    those filters a unit's weight is all that is needed, and
//                    the last workgroup draws;
//   k_sample_draw:   the tokens of those bins in a list, the weight above
//                    them by unit; the last workgroup of a row sorts the
//                    list, finds the cut and draws.
// A row whose list would not fit (thousands of tokens in one bin: equal
// logits) is cut by its first workgroup alone, digit by digit.
// Every sum is of whole numbers, so neither the order of the atomics nor the
// order of the list decides anything.
constexpr int kThreads = 256, kBlock = 8 * kThreads, kMaxSplits = 256, kUnits = kThreads, kBins = 512, kList = 4096;

struct alignas(128) RowWork {   // (whole lines)
  uint64_t unit[kUnits];         // weight kept for certain
  float top[kMaxSplits], low[kMaxSplits];
  uint32_t ticket[2], listed, done;   // done: 1 drawn, 2 cut by one workgroup
  // bins of the list: p0..p1 (top-p) and bk (top-k); kBins where that filter is off
  uint32_t p0, p1, bk, unused;
  uint64_t all;                       // weight of the row
  uint64_t count_p, weight_p, count_k, weight_k;   // before bin p0 and before bin bk
  // from here on only rows with top-k or top-p
  alignas(128) uint64_t weight[kBins];
  uint32_t count[kBins];
  uint64_t list[kList];          // (~key, index) of the tokens in the cut's bins: no more than the row's
};
// Bytes of a row's work; `filtered`: it may have top-k or top-p.
static int64_t row_work_bytes(int64_t V, bool filtered) {
  const int64_t list = 8 * (V < kList ? V : kList);
  const int64_t bytes = filtered ? (int64_t)offsetof(RowWork, list) + list : (int64_t)offsetof(RowWork, weight);
  return (bytes + 127) / 128 * 128;
}

struct SampleShared {
  uint64_t bins[kBins];          // count << 46 | weight
  uint64_t list[kList];
  uint64_t unit[kUnits];
  uint64_t part[kThreads / 64];
  float fpart[2][kThreads / 64];
  uint32_t cnt[256];
  uint64_t found[4];
  uint32_t pick[4];
  uint32_t last;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int by) {
  const uint32_t lo = __shfl_up((uint32_t)v, by), hi = __shfl_up((uint32_t)(v >> 32), by);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {   // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const uint64_t o = shfl_up64(v, by);
    if (lane >= by) v += o;
  }
  return v;
}
// Adds the lanes' values to *sum in LDS.
__device__ __forceinline__ void wave_add64(uint64_t* sum, uint64_t v) {
  if (!__ballot(v != 0)) return;
  v = wave_scan64(v);
  if ((threadIdx.x & 63) == 63) atomicAdd((unsigned long long*)sum, (unsigned long long)v);
}
// Exclusive prefix sum over the workgroup; `total` receives the sum.
__device__ __forceinline__ uint64_t block_scan64(SampleShared& s, uint64_t v, uint64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t inc = wave_scan64(v);
  __syncthreads();
  if (lane == 63) s.part[w] = inc;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const uint64_t p = s.part[i];
    if (i < w) before += p;
    total += p;
  }
  return before + inc - v;
}
__device__ __forceinline__ float block_max(float* part, float v) {
#pragma unroll
  for (int by = 32; by; by >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, by));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v = __builtin_fmaxf(v, part[i]);
  return v;
}

// The largest logit, and the smallest of those that are not far (where a
// weight is 0 for certain) below it, from each thread's own of both.  The
// second only sets the width of the bins.
struct Range { float top, low; };
__device__ __forceinline__ float far_of(const RowFilter& f) { return 32.0f / f.rate; }
__device__ __forceinline__ Range block_range(float (*part)[kThreads / 64], const RowFilter& f, float top, float low) {
  const float all = block_max(part[0], top);
  return Range{all, -block_max(part[1], all - low < far_of(f) ? -low : -__builtin_inff())};
}
// The row's range, and with it the bins: kBins of them down to the lowest
// logit, none wider than 1/16 of a power of two.
__device__ __forceinline__ void row_range(float (*part)[kThreads / 64], const RowWork& rw, int pieces, RowFilter& f) {
  const bool in = (int)threadIdx.x < pieces;
  const Range r = block_range(part, f, in ? rw.top[threadIdx.x] : -__builtin_inff(), in ? rw.low[threadIdx.x] : __builtin_inff());
  f.top = r.top;
  const float away = __builtin_fmaxf((r.top - r.low) * f.rate, 0x1p-20f);   // (a NaN where a row has no range)
  f.fine = __builtin_fmaxf((float)(kBins - 1) / away, kBins / 32.0f);
}

// Logits i .. i + 7 of a row, -inf past its end.  Rows of odd lengths start
// at any element: the 16-byte loads need not be aligned.
template <int DT>
__device__ __forceinline__ void load_logits(const void* row, int64_t i, int64_t V, float* v) {
  constexpr int kSize = DT == LOGITS_F32 ? 4 : 2;
  if (i + 8 <= V) {
    uint32_t w[2 * kSize];
    __builtin_memcpy(w, (const char*)row + i * kSize, 8 * kSize);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f;
      if constexpr (DT == LOGITS_F32) f = __builtin_bit_cast(float, w[j]);
      else if constexpr (DT == LOGITS_F16) f = h2f((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
      else f = __builtin_bit_cast(float, j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
      v[j] = no_nan(f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < V ? load_logit<DT>(row, i + j) : -__builtin_inff();
  }
}

__device__ __forceinline__ uint64_t place_of(float l, int64_t i) {   // ascending = sorted order
  return ((uint64_t)~order_key(l) << 32) | (uint32_t)i;
}

struct Piece { int64_t row; int64_t first, end; int piece; };
struct Split { int pieces; int64_t size; int units; int64_t unit, work; bool filtered; };   // `size` whole units; `work` bytes a row
__device__ __forceinline__ RowWork& work_of(RowWork* work, const Split& sp, int64_t row) {
  return *(RowWork*)((char*)work + row * sp.work);
}
__device__ __forceinline__ Piece my_piece(const Split& sp, int64_t V) {
  Piece p;
  const uint32_t row = blockIdx.x / (uint32_t)sp.pieces;   // (a 64-bit division would take longer than a short row)
  p.row = row;
  p.piece = (int)(blockIdx.x - row * (uint32_t)sp.pieces);
  p.first = p.piece * sp.size;
  p.end = p.first + sp.size < V ? p.first + sp.size : V;
  return p;
}
template <int DT>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int64_t row) {
  return (const char*)a.logits + row * a.ls * (DT == LOGITS_F32 ? 4 : 2);
}

// What the workgroups of a row hand to the last of them goes through
// device-scope atomics, which all XCDs see at one place.  (Plain stores and a
// device-wide fence per workgroup, which writes a whole L2 back, took 46 us
// for 600 workgroups that do 4 us of work.)
template <class T>
__device__ __forceinline__ void put(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T>
__device__ __forceinline__ T get(const T* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A piece's units, from the front of s.unit.
__device__ __forceinline__ void put_units(SampleShared& s, RowWork& rw, const Piece& p, const Split& sp) {
  const uint32_t unit = (uint32_t)sp.unit, first = (uint32_t)p.first / unit;   // (V is below 2^31)
  const int n = (int)(((uint32_t)(p.end - p.first) + unit - 1) / unit);
  __syncthreads();
  if ((int)threadIdx.x < n) put(&rw.unit[first + threadIdx.x], s.unit[threadIdx.x]);
}

// True in the workgroup that finishes its row's pass last: every workgroup
// counts itself once its atomics have completed.
__device__ __forceinline__ bool last_of_row(SampleShared& s, uint32_t* ticket, int pieces) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    s.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)pieces - 1;
  __syncthreads();
  return s.last;
}

__device__ __forceinline__ void put_token(const SampleArgs& a, int64_t row, const RowFilter& f, int64_t i, float l,
                                          uint64_t total) {
  a.ids[row] = i;
  a.logprobs[row] = -away_of(f, l) * 0x1.62e43p-1f - logf((float)total * 0x1p-31f);
}

// The draw, with the kept weight of each unit in s.unit: a token is kept
// when its place is at most `cut` and its weight at least f.least.
template <int DT>
__device__ void draw(SampleShared& s, const SampleArgs& a, const Split& sp, int64_t r, const RowFilter& f, uint64_t cut) {
  const int tid = threadIdx.x;
  const void* row = row_of<DT>(a, r);
  uint64_t total;
  const uint64_t mine = tid < sp.units ? s.unit[tid] : 0, before = block_scan64(s, mine, total);
  const double at = __builtin_floor((double)a.u[r] * (double)total);
  uint64_t target = at > 0.0 ? (uint64_t)at : 0;
  target = target < total ? target : total - 1;
  if (before <= target && target < before + mine) {
    s.pick[0] = tid;
    s.found[0] = target - before;
  }
  __syncthreads();
  const int unit = s.pick[0];
  uint64_t left = s.found[0];
  const int64_t end = (unit + 1) * sp.unit < a.V ? (unit + 1) * sp.unit : a.V;
  for (int64_t i0 = unit * sp.unit; i0 < end; i0 += kBlock) {
    const int64_t i = i0 + 8 * tid;
    float v[8];
    uint32_t w[8];
    load_logits<DT>(row, i, a.V, v);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = weight_of(f, v[j]);
      w[j] = w[j] >= f.least && place_of(v[j], i + j) <= cut ? w[j] : 0;
      sum += w[j];
    }
    uint64_t block;
    uint64_t run = block_scan64(s, sum, block);
    if (left < block) {
      if (run <= left && left < run + sum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (run <= left && left < run + w[j]) put_token(a, r, f, i + j, v[j], total);
          run += w[j];
        }
      }
      return;
    }
    left -= block;
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_top(SampleArgs a, Split sp, RowWork* work) {
  __shared__ float part[2][kThreads / 64];
  const Piece p = my_piece(sp, a.V);
  RowWork& rw = work_of(work, sp, p.row);
  if (sp.filtered)
    for (int i = p.piece * kThreads + threadIdx.x; i < kBins; i += sp.pieces * kThreads) {
      rw.weight[i] = 0;
      rw.count[i] = 0;
    }
  if (p.piece == 0 && threadIdx.x < 4) (&rw.ticket[0])[threadIdx.x] = 0;   // the tickets, listed and done
  const void* row = row_of<DT>(a, p.row);
  const RowFilter f = row_filter(a, p.row);
  const float far = far_of(f);
  const bool binned = f.k < a.V || f.p < 1.0;
  float top = -__builtin_inff(), low = __builtin_inff();
  for (int64_t i = p.first + 8 * threadIdx.x; i < p.end; i += kBlock) {
    float v[8];
    load_logits<DT>(row, i, a.V, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, v[j]);
    if (binned) {
      low = top - low < far ? low : top;   // what was low is far below by now
#pragma unroll
      for (int j = 0; j < 8; ++j) low = top - v[j] < far ? __builtin_fminf(low, v[j]) : low;
    }
  }
  const Range r = block_range(part, f, top, low);
  if (threadIdx.x == 0) {
    rw.top[p.piece] = r.top;
    rw.low[p.piece] = r.low;
  }
}

// In which bin a running sum over the bins reaches `target`: s.found = bin,
// count before it, weight before it.  Thread i holds bins 2 i and 2 i + 1.
template <bool BY_WEIGHT>
__device__ __forceinline__ void find_bin(SampleShared& s, uint64_t target, const uint64_t* n, const uint64_t* w,
                                         uint64_t nb, uint64_t wb) {
  __syncthreads();
  for (int j = 0; j < 2; ++j) {
    const uint64_t before = BY_WEIGHT ? wb : nb, size = BY_WEIGHT ? w[j] : n[j];
    if (before < target && target <= before + size) {
      s.found[0] = 2 * threadIdx.x + j;
      s.found[1] = nb;
      s.found[2] = wb;
      s.found[3] = BY_WEIGHT ? n[j] : w[j];
      s.pick[1] = (uint32_t)n[j];
    }
    nb += n[j];
    wb += w[j];
  }
  __syncthreads();
}

__device__ __forceinline__ uint64_t mass_of(double p, uint64_t all) {
  const double m = __builtin_ceil(p * (double)all);
  return m > 1.0 ? (uint64_t)m : 1;
}

// The bin of a token of any weight but 0; the last takes what the range left out.
__device__ __forceinline__ uint32_t bin_at(const RowFilter& f, float away) {
  return (uint32_t)__builtin_fminf(away * f.fine, (float)(kBins - 1));
}
__device__ __forceinline__ uint32_t bin_of(const RowFilter& f, float l) { return bin_at(f, away_of(f, l)); }

template <int DT>
__global__ __launch_bounds__(kThreads) void k_sample_bins(SampleArgs a, Split sp, RowWork* work) {
  __shared__ SampleShared s;
  const Piece p = my_piece(sp, a.V);
  RowWork& rw = work_of(work, sp, p.row);
  const int tid = threadIdx.x;
  const void* row = row_of<DT>(a, p.row);
  RowFilter f = row_filter(a, p.row);
  row_range(s.fpart, rw, sp.pieces, f);
  if (f.top == -__builtin_inff()) {   // every token masked
    if (p.piece == 0 && tid == 0) {
      a.ids[p.row] = -1;
      a.logprobs[p.row] = -__builtin_inff();
      rw.done = 1;
    }
    return;
  }
  const bool filtered = f.k < a.V || f.p < 1.0;
  if (!filtered) {
    s.unit[tid] = 0;
    __syncthreads();
    for (int64_t from = p.first, q = 0; from < p.end; from += sp.unit, ++q) {
      const int64_t to = from + sp.unit < p.end ? from + sp.unit : p.end;
      uint64_t sum = 0;
      for (int64_t i = from + 8 * tid; i < to; i += kBlock) {
        float v[8];
        load_logits<DT>(row, i, a.V, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w = weight_of(f, v[j]);
          sum += w >= f.least ? w : 0;
        }
      }
      wave_add64(&s.unit[q], sum);
    }
    put_units(s, rw, p, sp);
    if (!last_of_row(s, &rw.ticket[0], sp.pieces)) return;
    s.unit[tid] = tid < sp.units ? get(&rw.unit[tid]) : 0;
    if (tid == 0) rw.done = 1;
    __syncthreads();
    draw<DT>(s, a, sp, p.row, f, ~0ull);
    return;
  }
  // 2^14 tokens of at most 2^31 each at a time: 15 bits of count, 46 of weight
  for (int64_t from = p.first; from < p.end; from += 8 * kBlock) {
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
    __syncthreads();
    const int64_t to = from + 8 * kBlock < p.end ? from + 8 * kBlock : p.end;
    for (int64_t i = from + 8 * tid; i < to; i += kBlock) {
      float v[8];
      load_logits<DT>(row, i, a.V, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float away = away_of(f, v[j]);
        const uint32_t w = weight_at(away);
        if (w) atomicAdd((unsigned long long*)&s.bins[bin_at(f, away)], (1ull << 46) | w);
      }
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) {
      const uint64_t b = s.bins[i];
      if (b) {
        atomicAdd((unsigned long long*)&rw.weight[i], (unsigned long long)(b & ((1ull << 46) - 1)));
        atomicAdd(&rw.count[i], (uint32_t)(b >> 46));
      }
    }
    __syncthreads();
  }
  if (!last_of_row(s, &rw.ticket[0], sp.pieces)) return;
  uint64_t n[2], w[2], tokens, all;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    n[j] = get(&rw.count[2 * tid + j]);
    w[j] = get(&rw.weight[2 * tid + j]);
  }
  const uint64_t nb = block_scan64(s, n[0] + n[1], tokens), wb = block_scan64(s, w[0] + w[1], all);
  uint32_t bk = kBins, p0 = kBins, p1 = kBins;
  uint64_t count_p = 0, weight_p = 0, count_k = 0, weight_k = 0, low = all, high = all, listed = 0;
  if ((uint64_t)f.k < tokens) {
    find_bin<false>(s, f.k, n, w, nb, wb);
    bk = (uint32_t)s.found[0];
    count_k = s.found[1];
    weight_k = s.found[2];
    // the first tokens of the bin weigh at least their share of it
    const uint64_t in = s.found[3], size = s.pick[1], take = f.k - count_k;
    low = weight_k + (uint64_t)((double)in * ((double)take / (double)size) * (1.0 - 0x1p-40));
    high = weight_k + in;
    listed = size;
  }
  if (f.p < 1.0) {
    find_bin<true>(s, mass_of(f.p, high), n, w, nb, wb);
    p1 = (uint32_t)s.found[0];
    uint64_t in_p = s.pick[1];
    find_bin<true>(s, mass_of(f.p, low), n, w, nb, wb);
    p0 = (uint32_t)s.found[0];
    count_p = s.found[1];
    weight_p = s.found[2];
    if (p0 != p1 || bk <= p1) {   // tokens from p0 to p1, and bk's where it is not among them
      uint64_t in = 0, span;
      for (int j = 0; j < 2; ++j) {
        const uint32_t b = 2 * tid + j;
        if ((b >= p0 && b <= p1) || b == bk) in += n[j];
      }
      block_scan64(s, in, span);
      listed = span;
    } else {
      listed += in_p;
    }
  }
  if (tid == 0) {
    rw.bk = bk;
    rw.p0 = p0;
    rw.p1 = p1;
    rw.count_p = count_p;
    rw.weight_p = weight_p;
    rw.count_k = count_k;
    rw.weight_k = weight_k;
    rw.all = all;
    if (listed > kList) rw.done = 2;
  }
}

struct Place { uint64_t place, weight; };   // a token's place and the weight of the list before it

// The token of s.list, among those of bins b0..b1, at which the running count
// (BY_WEIGHT: weight) in the order of the places reaches `target`: up to 8
// bits at a time from the first that differs.  The target must be reached.
template <bool BY_WEIGHT>
__device__ Place select_place(SampleShared& s, uint32_t n, const RowFilter& f, uint32_t b0, uint32_t b1, uint64_t target) {
  const int tid = threadIdx.x;
  uint64_t* sum = s.bins;   // 256 weights
  auto takes = [&](uint64_t c) {
    if (b0 == 0 && b1 == (uint32_t)kBins) return true;
    const uint32_t b = bin_of(f, logit_of(~(uint32_t)(c >> 32)));
    return b >= b0 && b <= b1;
  };
  if (n <= 64) {   // every token counts those before it, each wave a quarter of them
    const uint32_t at = tid & 63, q = tid >> 6;
    const uint64_t e = at < n ? s.list[at] : 0;
    const uint32_t w = weight_of(f, logit_of(~(uint32_t)(e >> 32)));
    const bool in = at < n && takes(e);
    __syncthreads();
    if (q == 0) sum[at] = in ? w : 0;   // tokens that do not take part count nothing
    __syncthreads();
    uint64_t weight = 0;
    uint32_t count = 0;
    const uint32_t end = 16 * q + 16 < n ? 16 * q + 16 : n;
    for (uint32_t i = 16 * q; i < end; ++i) {
      const uint64_t wi = s.list[i] < e ? sum[i] : 0;
      count += wi != 0;
      weight += wi;
    }
    sum[64 + tid] = weight;
    s.cnt[tid] = count;
    __syncthreads();
    if (q == 0 && in) {
      weight = sum[64 + at] + sum[128 + at] + sum[192 + at] + sum[256 + at];
      count = s.cnt[at] + s.cnt[64 + at] + s.cnt[128 + at] + s.cnt[192 + at];
      if (BY_WEIGHT ? weight < target && target <= weight + w : count + 1 == target) {
        s.found[0] = e;
        s.found[2] = weight;
      }
    }
    __syncthreads();
    const Place c{s.found[0], s.found[2]};
    __syncthreads();
    return c;
  }
  uint64_t any = 0, each = ~0ull;
  for (uint32_t i = tid; i < n; i += kThreads)
    if (takes(s.list[i])) {
      any |= s.list[i];
      each &= s.list[i];
    }
#pragma unroll
  for (int by = 32; by; by >>= 1) {
    any |= ((uint64_t)(uint32_t)__shfl_xor((int)(any >> 32), by) << 32) | (uint32_t)__shfl_xor((int)any, by);
    each &= ((uint64_t)(uint32_t)__shfl_xor((int)(each >> 32), by) << 32) | (uint32_t)__shfl_xor((int)each, by);
  }
  __syncthreads();
  if ((tid & 63) == 0) {
    s.part[tid >> 6] = any;
    s.found[tid >> 6] = each;
  }
  __syncthreads();
  any = s.part[0] | s.part[1] | s.part[2] | s.part[3];
  each = s.found[0] & s.found[1] & s.found[2] & s.found[3];
  Place c{each, 0};
  uint64_t count = 0;
  // from the highest bit that differs, up to 8 bits at a time
  int top = any == each ? 0 : 64 - __builtin_clzll(any ^ each), shift;
  if (top) c.place = top == 64 ? 0 : each >> top << top;   // what all share
  for (; top; top = shift) {
    shift = top > 8 ? top - 8 : 0;
    const uint32_t mask = (1u << (top - shift)) - 1;
    __syncthreads();
    s.cnt[tid] = 0;
    sum[tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kThreads) {
      const uint64_t e = s.list[i];
      if (takes(e) && (top == 64 || (e >> top) == (c.place >> top))) {
        const uint32_t digit = (uint32_t)(e >> shift) & mask;
        atomicAdd(&s.cnt[digit], 1u);
        atomicAdd((unsigned long long*)&sum[digit], (unsigned long long)weight_of(f, logit_of(~(uint32_t)(e >> 32))));
      }
    }
    __syncthreads();
    if (tid < 64) {   // lane i: digits 4 i to 4 i + 3
      uint64_t nn = 0, ww = 0;
      for (int j = 0; j < 4; ++j) {
        nn += s.cnt[4 * tid + j];
        ww += sum[4 * tid + j];
      }
      uint64_t nb = count + wave_scan64(nn) - nn, wb = c.weight + wave_scan64(ww) - ww;
      for (int j = 0; j < 4; ++j) {
        const uint64_t ne = nb + s.cnt[4 * tid + j], we = wb + sum[4 * tid + j];
        if (BY_WEIGHT ? wb < target && target <= we : nb < target && target <= ne) {
          s.found[0] = 4 * tid + j;
          s.found[1] = nb;
          s.found[2] = wb;
          s.found[3] = ne - nb;
        }
        nb = ne;
        wb = we;
      }
    }
    __syncthreads();
    c.place |= s.found[0] << shift;
    count = s.found[1];
    c.weight = s.found[2];
    if (s.found[3] == 1) {   // one token has these digits
      __syncthreads();
      for (uint32_t i = tid; i < n; i += kThreads)
        if (takes(s.list[i]) && (s.list[i] >> shift) == (c.place >> shift)) s.found[0] = s.list[i];
      __syncthreads();
      c.place = s.found[0];
      break;
    }
  }
  __syncthreads();
  return c;
}

struct Cut { uint32_t key; uint64_t count, weight; };   // tokens and weight before the key's first one

// The bits that any and that all of the row's keys have, tokens of weight 0 aside.
struct KeyBits { uint32_t any, each; };
template <int DT>
__device__ KeyBits key_bits(SampleShared& s, const void* row, int64_t V, const RowFilter& f) {
  uint32_t any = 0, each = ~0u;
#pragma unroll 4
  for (int64_t i = 8 * threadIdx.x; i < V; i += kBlock) {
    float v[8];
    load_logits<DT>(row, i, V, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t key = order_key(v[j]);
      const bool in = weight_of(f, v[j]) != 0;
      any |= in ? key : 0;
      each &= in ? key : ~0u;
    }
  }
#pragma unroll
  for (int by = 32; by; by >>= 1) {
    any |= (uint32_t)__shfl_xor((int)any, by);
    each &= (uint32_t)__shfl_xor((int)each, by);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = ((uint64_t)any << 32) | each;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    any |= (uint32_t)(s.part[i] >> 32);
    each &= (uint32_t)s.part[i];
  }
  return KeyBits{any, each};
}

// The key at which the sorted row's running count (BY_WEIGHT: weight) reaches
// `target`, up to 8 bits at a time from the first that differs; tokens of
// weight 0 do not count.  The target must be reached.
template <int DT, bool BY_WEIGHT>
__device__ Cut select_key(SampleShared& s, const void* row, int64_t V, const RowFilter& f, KeyBits bits, uint64_t target) {
  Cut c{bits.each, 0, 0};
  uint64_t* sum = s.list;
  int top = bits.any == bits.each ? 0 : 32 - __builtin_clz(bits.any ^ bits.each), shift;
  if (top) c.key = top == 32 ? 0 : bits.each >> top << top;   // what all share
  for (; top; top = shift) {
    shift = top > 8 ? top - 8 : 0;
    const uint32_t mask = (1u << (top - shift)) - 1;
    __syncthreads();
    s.cnt[threadIdx.x] = 0;
    sum[threadIdx.x] = 0;
    __syncthreads();
    // (whole waves step together: the last block's lanes past the row load nothing)
    for (int64_t i0 = 0; i0 < V; i0 += kBlock) {
      const int64_t i = i0 + 8 * threadIdx.x;
      float v[8];
      load_logits<DT>(row, i, V, v);
      uint32_t w[8], digit[8];
      int mine = -1;
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        const uint32_t key = order_key(v[j]);
        w[j] = top == 32 || (key >> top) == (c.key >> top) ? weight_of(f, v[j]) : 0;
        digit[j] = (key >> shift) & mask;
        mine = w[j] ? (int)digit[j] : mine;
      }
      // equal logits would queue at one counter: the wave's tokens of one digit go together
      const uint64_t with = __ballot(mine >= 0);
      if (!with) continue;
      const uint32_t lead = (uint32_t)__builtin_amdgcn_readlane(mine, __builtin_ctzll(with));
      uint64_t together = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w[j]) {
          if (digit[j] == lead) {
            together += (1ull << 46) | w[j];
          } else {
            atomicAdd(&s.cnt[digit[j]], 1u);
            atomicAdd((unsigned long long*)&sum[digit[j]], (unsigned long long)w[j]);
          }
        }
      together = wave_scan64(together);
      if ((threadIdx.x & 63) == 63) {
        atomicAdd(&s.cnt[lead], (uint32_t)(together >> 46));
        atomicAdd((unsigned long long*)&sum[lead], (unsigned long long)(together & ((1ull << 46) - 1)));
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {   // lane i: digits 255 - 4 i down to 252 - 4 i
      const int d0 = 255 - 4 * (int)threadIdx.x;
      uint64_t n = 0, w = 0;
      for (int j = 0; j < 4; ++j) {
        n += s.cnt[d0 - j];
        w += sum[d0 - j];
      }
      uint64_t nb = c.count + wave_scan64(n) - n, wb = c.weight + wave_scan64(w) - w;
      for (int j = 0; j < 4; ++j) {
        const uint64_t nn = nb + s.cnt[d0 - j], ww = wb + sum[d0 - j];
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

// The cut of a whole row by one workgroup, for rows of many equal logits.
template <int DT>
__device__ uint64_t cut_row(SampleShared& s, const RowWork& rw, const void* row, int64_t V, const RowFilter& f) {
  uint32_t key = 0;
  uint64_t ties = 0, all = rw.all;
  const KeyBits bits = key_bits<DT>(s, row, V, f);
  if (rw.bk < (uint32_t)kBins) {
    const Cut c = select_key<DT, false>(s, row, V, f, bits, f.k);
    key = c.key;
    ties = f.k - c.count;
    all = c.weight + ties * weight_of(f, logit_of(key));
  }
  if (f.p < 1.0) {   // at or above the top-k cut: the mass is at most all
    const uint64_t mass = mass_of(f.p, all);
    const Cut c = select_key<DT, true>(s, row, V, f, bits, mass);
    const uint64_t each = weight_of(f, logit_of(c.key));
    key = c.key;
    ties = (mass - c.weight + each - 1) / each;
  }
  // the index of the last of the key's `ties` first tokens
  __syncthreads();
  if (threadIdx.x == 0) s.found[0] = 0xffffffffu;
  constexpr int kWide = 2;   // blocks at a time
  for (int64_t i0 = 0; i0 < V; i0 += kWide * kBlock) {
    const int64_t i = i0 + 8 * kWide * threadIdx.x;
    float v[8 * kWide];
#pragma unroll
    for (int q = 0; q < kWide; ++q) load_logits<DT>(row, i + 8 * q, V, v + 8 * q);
    uint64_t n = 0, block;
#pragma unroll
    for (int j = 0; j < 8 * kWide; ++j) n += i + j < V && order_key(v[j]) == key;
    uint64_t run = block_scan64(s, n, block);
    if (ties <= block) {
#pragma unroll
      for (int j = 0; j < 8 * kWide; ++j) {
        const bool in = i + j < V && order_key(v[j]) == key;
        run += in;
        if (in && run == ties) s.found[0] = (uint32_t)(i + j);
      }
      break;
    }
    ties -= block;
  }
  __syncthreads();
  return ((uint64_t)~key << 32) | (uint32_t)s.found[0];
}

template <int DT>
__global__ __launch_bounds__(kThreads, 4) void k_sample_draw(SampleArgs a, Split sp, RowWork* work) {
  __shared__ SampleShared s;
  const Piece p = my_piece(sp, a.V);
  RowWork& rw = work_of(work, sp, p.row);
  const int tid = threadIdx.x;
  const uint32_t done = rw.done;
  if (done == 1 || (done == 2 && p.piece)) return;
  const void* row = row_of<DT>(a, p.row);
  RowFilter f = row_filter(a, p.row);
  row_range(s.fpart, rw, sp.pieces, f);
  const uint32_t p0 = rw.p0, p1 = rw.p1, bk = rw.bk;
  if (done == 2) {
    const uint64_t cut = cut_row<DT>(s, rw, row, a.V, f);
    __syncthreads();
    s.unit[tid] = 0;
    __syncthreads();
    for (int q = tid >> 6; q < sp.units; q += kThreads / 64) {   // a unit for each wave
      const int64_t first = q * sp.unit, end = first + sp.unit < a.V ? first + sp.unit : a.V;
      uint64_t sum = 0;
#pragma unroll 4
      for (int64_t i = first + 8 * (tid & 63); i < end; i += 512) {
        float v[8];
        load_logits<DT>(row, i, a.V, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w = weight_of(f, v[j]);
          sum += w >= f.least && place_of(v[j], i + j) <= cut ? w : 0;
        }
      }
      wave_add64(&s.unit[q], sum);
    }
    __syncthreads();
    draw<DT>(s, a, sp, p.row, f, cut);
    return;
  }

  // weight above the cut's first bin, and the tokens of the cut's bins
  const uint32_t above = p0 < (uint32_t)kBins ? p0 : bk, end = bk < (uint32_t)kBins ? bk + 1 : p1 + 1;
  const float above_f = (float)above, end_f = (float)end;
  if (tid == 0) s.pick[0] = 0;
  s.unit[tid] = 0;
  __syncthreads();
  for (int64_t from = p.first, q = 0; from < p.end; from += sp.unit, ++q) {
    const int64_t to = from + sp.unit < p.end ? from + sp.unit : p.end;
    uint64_t sum = 0;
    for (int64_t i = from + 8 * tid; i < to; i += kBlock) {
      float v[8];
      load_logits<DT>(row, i, a.V, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float away = away_of(f, v[j]), t = __builtin_fminf(away * f.fine, (float)(kBins - 1));
        if (t < end_f) {   // few tokens, and few waves that hold one
          const uint32_t w = weight_at(away), b = (uint32_t)t;
          if (t < above_f) sum += w >= f.least ? w : 0;
          else if (w && ((p0 <= b && b <= p1) || b == bk)) s.list[atomicAdd(&s.pick[0], 1u)] = place_of(v[j], i + j);
        }
      }
    }
    wave_add64(&s.unit[q], sum);
  }
  put_units(s, rw, p, sp);   // (the list is complete, too)
  const uint32_t mine = s.pick[0];
  if (tid == 0) s.pick[1] = mine ? atomicAdd(&rw.listed, mine) : 0;
  __syncthreads();
  for (uint32_t i = tid; i < mine; i += kThreads) put(&rw.list[s.pick[1] + i], s.list[i]);
  if (!last_of_row(s, &rw.ticket[1], sp.pieces)) return;

  const uint32_t n = get(&rw.listed);
  for (uint32_t i = tid; i < n; i += kThreads) s.list[i] = get(&rw.list[i]);
  __syncthreads();
  // Bins that do not touch are two runs of the sorted row, each with its own
  // count and weight before it; top-p ends in the first, top-k in the second.
  const bool with_k = bk < (uint32_t)kBins, with_p = p0 < (uint32_t)kBins, two = with_k && with_p && p1 + 1 < bk;
  const uint64_t first_k = two || !with_p ? rw.count_k : rw.count_p, weight_k = two || !with_p ? rw.weight_k : rw.weight_p;
  uint64_t all = rw.all, cut = ~0ull;
  if (with_k) {
    const Place c = select_place<false>(s, n, f, two ? bk : 0, kBins, (uint64_t)f.k - first_k);
    cut = c.place;
    all = weight_k + c.weight + weight_of(f, logit_of(~(uint32_t)(cut >> 32)));
  }
  if (with_p) cut = select_place<true>(s, n, f, 0, two ? p1 : kBins, mass_of(f.p, all) - rw.weight_p).place;
  const uint32_t per = (n + kThreads - 1) / kThreads, i0 = tid * per < n ? tid * per : n, i1 = i0 + per < n ? i0 + per : n;
  __syncthreads();
  s.unit[tid] = tid < sp.units ? get(&rw.unit[tid]) : 0;
  __syncthreads();
  for (uint32_t i = i0; i < i1; ++i)
    if (s.list[i] <= cut) {
      const uint32_t w = weight_of(f, logit_of(~(uint32_t)(s.list[i] >> 32)));
      if (w >= f.least) atomicAdd((unsigned long long*)&s.unit[(uint32_t)s.list[i] / (uint32_t)sp.unit], (unsigned long long)w);
    }
  __syncthreads();
  draw<DT>(s, a, sp, p.row, f, cut);
}

// Pieces of at least one unit, so many that the rows together
// make about four workgroups a compute unit.
static Split sample_split(int64_t batch, int64_t V) {
  const int64_t blocks = (V + kBlock - 1) / kBlock, unit = (blocks + kUnits - 1) / kUnits, all = (blocks + unit - 1) / unit;
  int64_t pieces = 1024 / (batch < 1024 ? batch : 1024);
  pieces = pieces < 1 ? 1 : pieces;
  pieces = pieces < all ? pieces : all;
  pieces = pieces < kMaxSplits ? pieces : kMaxSplits;
  const int64_t per = (all + pieces - 1) / pieces;
  return Split{(int)((all + per - 1) / per), per * unit * kBlock, (int)all, unit * kBlock, 0, false};
}

// Whether a row can have top-k or top-p (a temperature of 0 is a top-k of 1).
static bool sample_filtered(bool per_row, int64_t V, float temperature, int32_t top_k, float top_p) {
  return per_row || !(temperature > 0.f) || (top_k > 0 && top_k < V) || top_p < 1.f;
}

template <int DT>
static void launch_sample(const SampleArgs& a, const Split& sp, RowWork* work, hipStream_t stream) {
  const dim3 grid((unsigned)(a.batch * sp.pieces)), block(kThreads);
  hipLaunchKernelGGL(k_sample_top<DT>, grid, block, 0, stream, a, sp, work);
  hipLaunchKernelGGL(k_sample_bins<DT>, grid, block, 0, stream, a, sp, work);
  // where no row can have top-k or top-p the second launch has drawn them all
  if (sp.filtered) hipLaunchKernelGGL(k_sample_draw<DT>, grid, block, 0, stream, a, sp, work);
}

}  // namespace m2r

using namespace m2r;

extern "C" int64_t m2r_sample_workspace(int64_t batch, int64_t V) {
  return batch > 0 && V > 0 ? batch * row_work_bytes(V, true) : 0;
}

extern "C" int64_t m2r_sample_call_workspace(int64_t batch, int64_t V, int per_row, float temperature_all,
                                             int32_t top_k_all, float top_p_all) {
  if (batch <= 0 || V <= 0) return 0;
  return batch * row_work_bytes(V, sample_filtered(per_row, V, temperature_all, top_k_all, top_p_all));
}

extern "C" int m2r_sample(const void* logits, int dtype, int64_t row_stride, const float* uniforms,
                          const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                          const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* ids,
                          float* logprobs, int64_t batch, int64_t V, void* workspace, int64_t workspace_bytes,
                          hipStream_t stream) {
  if (batch <= 0 || V <= 0) return m2r_fail("sample: non-positive shape");
  if (batch > 0x7fffffff || V > 0x7fffffff) return m2r_fail("sample: size limits");
  if (dtype < LOGITS_F16 || dtype > LOGITS_F32) return m2r_fail("sample: logits must be binary16 (0), bfloat16 (1) or binary32 (2)");
  if (!logits || !uniforms || !ids || !logprobs) return m2r_fail("sample: null pointer");
  if (row_stride < V && batch > 1) return m2r_fail("sample: rows overlap");
  SampleArgs a{logits, row_stride, uniforms, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all,
               top_k_all, ids, logprobs, batch, V};
  const bool filtered = sample_filtered(temperature || top_k || top_p, V, temperature_all, top_k_all, top_p_all);
  Split sp = sample_split(batch, V);
  sp.work = row_work_bytes(V, filtered);
  sp.filtered = filtered;
  if (!workspace || workspace_bytes < batch * sp.work || ((uintptr_t)workspace & 15))
    return m2r_fail("sample: workspace too small or not 16-byte aligned");
  if (batch * sp.pieces > 0x7fffffff) return m2r_fail("sample: grid limits exceeded");
  RowWork* work = (RowWork*)workspace;
  if (dtype == LOGITS_F16) launch_sample<LOGITS_F16>(a, sp, work, stream);
  else if (dtype == LOGITS_BF16) launch_sample<LOGITS_BF16>(a, sp, work, stream);
  else launch_sample<LOGITS_F32>(a, sp, work, stream);
  return m2r_check(hipGetLastError(), "sample launch");
}
