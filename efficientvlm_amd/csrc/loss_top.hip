// Distillation from a teacher's TOP logits for gfx950: the k largest logits of every row with their classes and the row's
// log-sum-exp (what a teacher that ran ahead, or offline, keeps of a row of tens of thousands of classes), the loss against
// a student's whole rows and its gradient.  f32 and bf16 logits, everything else f32.
//
//   y = student logits / T,  q = softmax(y) over all C classes,  z_j = kept teacher logits / T of the classes i_j
//   without the teacher's lse:  p = softmax(z) over the kept classes,        L_r = sum_j p_j (log p_j - log q_{i_j})
//   with it:  p_j = exp(z_j - lse_t),  p_rest = 1 - sum_j p_j,               L_r += p_rest (log p_rest - log q_rest),
//             q_rest = the student's mass on the classes that are not kept (one class more for both)
//   loss = sum_r w_r L_r / R
//   d L_r / d y_c = M q_c - sum_{j: i_j = c} p_j            kept classes       (M = sum_j p_j + p_rest, 1 up to rounding)
//                 = q_c / q_rest (M q_rest - p_rest)         all others, with a rest;  M q_c without
//   An entry whose class lies outside [0, C) takes no part; a row without entries adds nothing and has a zero gradient.
//
// All three kernels stream rows: one workgroup per row, 16-byte loads (rows need not be 16-byte aligned: the hardware takes
// any alignment), sums in f32 in a fixed order.
#include "common.h"

#define TOP_MAX_K 256
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// 8 consecutive elements of a row from any element-aligned address
template <typename T> __device__ __forceinline__ void load8_any(const T* p, float v[8]);
template <> __device__ __forceinline__ void load8_any<bf16>(const bf16* p, float v[8]) {
  bf16x8 t;
  __builtin_memcpy(&t, p, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
template <> __device__ __forceinline__ void load8_any<float>(const float* p, float v[8]) {
  f32x4 t[2];
  __builtin_memcpy(t, p, 32);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = t[i >> 2][i & 3];
}
// elements 8c .. 8c + 7 of a row of C; `fill` behind its end
template <typename T> __device__ __forceinline__ void row8(const T* x, int c, int C, float fill, float v[8]) {
  if (8 * c + 8 <= C) { load8_any<T>(x + 8 * (int64_t)c, v); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 8 * c + e < C ? to_f(x[8 * (int64_t)c + e]) : fill;
}

// the same 8 elements as they are stored, to be kept in registers between sweeps
template <typename T> struct TopRaw8;
template <> struct TopRaw8<bf16> {
  bf16x8 t;
  __device__ __forceinline__ void get(float v[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  }
  __device__ __forceinline__ void set(int i, bf16 x) { t[i] = x; }
  __device__ __forceinline__ void drop(uint32_t bits) {      // -inf where the bit is set (a select by masks: 4 instructions a pair)
    uint32_t w[4];
    __builtin_memcpy(w, &t, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = __builtin_amdgcn_sbfe((int)bits, 2 * i, 1), hi = __builtin_amdgcn_sbfe((int)bits, 2 * i + 1, 1);
      const uint32_t mask = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
      w[i] = (mask & 0xFF80FF80u) | (~mask & w[i]);
    }
    __builtin_memcpy(&t, w, 16);
  }
};
template <> struct TopRaw8<float> {
  f32x4 t[2];
  __device__ __forceinline__ void get(float v[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = t[i >> 2][i & 3];
  }
  __device__ __forceinline__ void set(int i, float x) { t[i >> 2][i & 3] = x; }
  __device__ __forceinline__ void drop(uint32_t bits) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i >> 2][i & 3] = (bits >> i) & 1u ? -INFINITY : t[i >> 2][i & 3];
  }
};
template <typename T> __device__ __forceinline__ void raw8(const T* x, int c, int C, float fill, TopRaw8<T>& o) {
  if (8 * c + 8 <= C) { __builtin_memcpy(&o, x + 8 * (int64_t)c, sizeof(o)); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) o.set(e, 8 * c + e < C ? x[8 * (int64_t)c + e] : from_f<T>(fill));
}

// ---------------------------------------------------------------------------------------------
// the k largest logits of a row
// ---------------------------------------------------------------------------------------------
// order-preserving key of a float: NaN above everything, -0 = +0; 0 is below every value
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int block_count(int v, int* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < nw; ++i) t += red[i];
  return t;
}

// One sweep finds every thread's own maximum; the k-th largest of those maxima (its upper 16 bits: a bisection by one wave) is
// a lower bound of the k-th largest element, and barely more than k elements reach it.  Those are collected and ranked by
// counting, (value, lower class first) making every element distinct - the result does not depend on the order of collection.
// Rows with long ties at the bound (more candidates than the list holds) and rows with NaN or without a finite maximum get the
// exact bound by bisection over the row, first of the value, then of the class among equals.
// Bound by its vector instructions beside HBM: 8 elements cost 14 instructions for the maximum (which is kept) and 40 slots for the sum (an
// exponential takes two); the candidates are collected by pieces of 8 first (one compare a piece), then one element a thread: with every
// thread testing the 8 of its own pieces, a wave went through nearly all of them for two or three candidates.
// 3000 bf16 rows of 30 522, k = 64: 44 us = 4.2 TB/s (56 before these three); 7 rows: 7.8 us, the phases of one row after the other.
#define TOP_NT 512
#define TOP_CAP 1024
#define TOP_LOG2E 1.44269504088896341f
__device__ __forceinline__ float max8(const float (&v)[8]) {
  return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
__device__ __forceinline__ float max8(const TopRaw8<float>& x) {
  float v[8];
  x.get(v);
  return max8(v);
}
// bf16: their patterns two at a time.  As signed numbers the patterns of positive values are in order and above those of negative ones; among
// negative ones the smallest unsigned pattern is the largest value.  (14 instructions for the 8, where as floats - each is
// quieted first - they took 32.  A NaN may win or not: the sum of its row is NaN, and nothing is done with the maximum.)
__device__ __forceinline__ float max8(const TopRaw8<bf16>& x) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  uint32_t w[4];
  __builtin_memcpy(w, &x.t, 16);
  s16x2 hi = __builtin_bit_cast(s16x2, w[0]);
  u16x2 lo = __builtin_bit_cast(u16x2, w[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s16x2, w[i]));
    lo = __builtin_elementwise_min(lo, __builtin_bit_cast(u16x2, w[i]));
  }
  const int h = hi[0] > hi[1] ? hi[0] : hi[1];
  const unsigned l = lo[0] < lo[1] ? lo[0] : lo[1];
  return __uint_as_float((h >= 0 ? (unsigned)h : l) << 16);
}
// exp((v - m) / T) = 2^((v - m) c2), c2 = log2e / T
__device__ __forceinline__ float exp_diff(float v, float m, float c2) { return __builtin_amdgcn_exp2f((v - m) * c2); }
// Sums of it over a row: v c2 - m c2 in one fma, and the sum afterwards by what the rounding of m c2 left (tail), so that it is as exact as
// with the difference first.  That rounding is half a unit of m c2, at most 1/2 up to 2^24; from 2^31 on it alone would take the terms
// out of range (a maximum of -1e10, as masks leave it), so beyond 2^24 the difference comes first.
struct ExpSum {
  float m, c2, off;
  bool in_range;
  __device__ __forceinline__ ExpSum(float m_, float c2_) : m(m_), c2(c2_), off(-m_ * c2_), in_range(fabsf(m_ * c2_) <= 0x1p24f) {}
  __device__ __forceinline__ float tail() const { return in_range ? __builtin_amdgcn_exp2f(-fmaf(m, c2, off)) : 1.0f; }
  template <bool FAST> __device__ __forceinline__ float of(float v) const {
    return FAST ? __builtin_amdgcn_exp2f(fmaf(v, c2, off)) : exp_diff(v, m, c2);
  }
};
template <typename T, int NCH>
__global__ __launch_bounds__(TOP_NT, sizeof(T) == 2 ? 8 : 4) void top_logits_kernel(const T* __restrict__ logits, int C, int64_t ld, int k, float inv_t,
                                                            float* __restrict__ values, int32_t* __restrict__ classes,
                                                            float* __restrict__ lse) {
  __shared__ float red[16];
  __shared__ int ired[16];
  __shared__ uint32_t tops[TOP_NT];
  __shared__ unsigned long long list[TOP_CAP];
  __shared__ uint32_t hits[TOP_CAP];
  __shared__ uint32_t bound;
  __shared__ int count, nhits;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t r = blockIdx.x;
  const T* x = logits + r * ld;
  const int chunks = (C + 7) >> 3;
  // rows of up to NCH * 8 * TOP_NT elements stay in registers between the sweeps (NCH = 0: longer ones are read again)
  TopRaw8<T> keep[NCH > 0 ? NCH : 1];
  float most[NCH > 0 ? NCH : 1];                             // maximum of each 8
  if constexpr (NCH > 0) {
#pragma unroll
    for (int n = 0; n < NCH; ++n)
      if (tid + n * TOP_NT < chunks) raw8<T>(x, tid + n * TOP_NT, C, -INFINITY, keep[n]);
  }
  auto again = [&](auto f) __attribute__((always_inline)) {
    for (int c = tid; c < chunks; c += TOP_NT) {
      float v[8];
      row8<T>(x, c, C, -INFINITY, v);
      f(v, 8 * c);
    }
  };
  float mx = -INFINITY;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      most[n] = -INFINITY;
      if (tid + n * TOP_NT < chunks) {
        most[n] = max8(keep[n]);
        mx = fmaxf(mx, most[n]);
      }
    }
  } else {
    again([&](const float (&v)[8], int) { mx = fmaxf(mx, max8(v)); });
  }
  tops[tid] = tid < chunks ? order_key(mx) : 0u;
  if (tid == 0) { count = 0; nhits = 0; }
  const float M = block_max(mx, red);                        // (ends the hand-over of tops and count, too)
  if (tid < 64) {
    uint32_t t[TOP_NT / 64], b = 0;
#pragma unroll
    for (int j = 0; j < TOP_NT / 64; ++j) t[j] = tops[lane + 64 * j];
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t cand = b | (1u << bit);
      int n = 0;
#pragma unroll
      for (int j = 0; j < TOP_NT / 64; ++j) n += __popcll(__ballot(t[j] >= cand));
      if (n >= k) b = cand;
    }
    if (lane == 0) bound = b;
  }
  // sum of exp((v - M) / T): NaN where the row holds one, or has no finite maximum
  const ExpSum ex(M, inv_t * TOP_LOG2E);
  float s = 0.f;
  auto sweep = [&](auto fast) __attribute__((always_inline)) {
    auto add8 = [&](const float (&v)[8], int) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s += ex.template of<decltype(fast)::value>(v[e]);
    };
    if constexpr (NCH > 0) {
#pragma unroll
      for (int n = 0; n < NCH; ++n)
        if (tid + n * TOP_NT < chunks) {
          float v[8];
          keep[n].get(v);
          add8(v, 0);
        }
    } else {
      again(add8);
    }
  };
  if (ex.in_range) sweep(Yes()); else sweep(No());           // (block-uniform)
  s = block_sum(s, red) * ex.tail();
  const bool regular = s < INFINITY;                         // (block-uniform; false for NaN)
  if (regular) {
    if (tid == 0) lse[r] = M * inv_t + logf(s);
    const float b = key_value(max(bound, 0x00800000u));      // (the lowest finite value at least)
    // the pieces of 8 that hold a candidate, then their elements, one a thread (asked for again: few)
    auto hit = [&](int c) __attribute__((always_inline)) {
      const int at = atomicAdd(&nhits, 1);
      if (at < TOP_CAP) hits[at] = c;
    };
    if constexpr (NCH > 0) {
#pragma unroll
      for (int n = 0; n < NCH; ++n)
        if (most[n] >= b) hit(tid + n * TOP_NT);
    } else {
      again([&](const float (&v)[8], int i0) { if (max8(v) >= b) hit(i0 >> 3); });
    }
    __syncthreads();
    const int pieces = nhits;
    if (pieces > TOP_CAP) { if (tid == 0) count = TOP_CAP + 1; }
    else
      for (int i = tid; i < 8 * pieces; i += TOP_NT) {
        const int e = 8 * (int)hits[i >> 3] + (i & 7);
        if (e < C) {
          const float v = to_f(x[e]);
          if (v >= b) {
            const int at = atomicAdd(&count, 1);
            if (at < TOP_CAP) list[at] = ((unsigned long long)order_key(v) << 32) | (uint32_t)~e;
          }
        }
      }
  } else {
    int nan = 0;
    again([&](const float (&v)[8], int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) nan |= v[e] != v[e] ? 1 : 0;
    });
    const bool bad = block_count(nan, ired) != 0;
    if (tid == 0) lse[r] = bad ? __builtin_nanf("") : M;
  }
  __syncthreads();
  int n = regular && count >= k ? count : TOP_CAP + 1;       // (fewer than k finite ones: -inf has to be chosen among, too)
  if (n > TOP_CAP) {                                         // (block-uniform)
    auto reach = [&](uint32_t lo) {                          // elements with a key >= lo
      int m = 0;
      again([&](const float (&v)[8], int i0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m += (order_key(v[e]) >= lo && i0 + e < C) ? 1 : 0;
      });
      return block_count(m, ired);
    };
    uint32_t v0 = 0;                                         // largest key that at least k elements reach
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = v0 | (1u << bit);
      if (reach(cand) >= k) v0 = cand;
    }
    const int more = v0 == 0xFFFFFFFFu ? 0 : reach(v0 + 1), need = k - more;      // `need` of the elements equal to v0
    int lo = 0, hi = C;                                      // smallest hi with need equal elements below it
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      int m = 0;
      again([&](const float (&v)[8], int i0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m += (order_key(v[e]) == v0 && i0 + e < mid && i0 + e < C) ? 1 : 0;
      });
      if (block_count(m, ired) >= need) hi = mid; else lo = mid + 1;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    again([&](const float (&v)[8], int i0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = order_key(v[e]);
        if (i0 + e < C && (key > v0 || (key == v0 && i0 + e < hi))) {
          const int at = atomicAdd(&count, 1);
          if (at < TOP_CAP) list[at] = ((unsigned long long)key << 32) | (uint32_t)~(i0 + e);
        }
      }
    });
    __syncthreads();
    n = min(count, TOP_CAP);
  }
  for (int i = tid; i < n; i += TOP_NT) {
    const unsigned long long mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > mine ? 1 : 0;
    if (rank < k) {
      values[r * k + rank] = key_value((uint32_t)(mine >> 32));
      classes[r * k + rank] = (int32_t)~(uint32_t)mine;
    }
  }
}

extern "C" int evlm_top_logits(int dtype, const void* logits, int R, int C, int64_t ld, int k, float inv_t, float* values,
                               int32_t* classes, float* lse, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  EVLM_REQUIRE(logits && values && classes && lse && R > 0 && C > 0 && ld >= C, "evlm_top_logits: bad args");
  EVLM_REQUIRE(k > 0 && k <= TOP_MAX_K && k <= C, "evlm_top_logits: k = %d is not in 1 .. min(%d, classes)", k, TOP_MAX_K);
  EVLM_REQUIRE(C <= (1 << 30), "evlm_top_logits: too many classes");
  EVLM_REQUIRE(inv_t > 0.f && inv_t < 1e30f, "evlm_top_logits: the temperature must be positive and finite");
  EVLM_DISPATCH_DTYPE(dtype, "evlm_top_logits",
    if (C <= 8 * 8 * TOP_NT)
      hipLaunchKernelGGL((top_logits_kernel<T, 8>), dim3(R), dim3(TOP_NT), 0, stream, (const T*)logits, C, ld, k, inv_t, values, classes, lse);
    else
      hipLaunchKernelGGL((top_logits_kernel<T, 0>), dim3(R), dim3(TOP_NT), 0, stream, (const T*)logits, C, ld, k, inv_t, values, classes, lse);)
  EVLM_LAUNCH_CHECK("evlm_top_logits");
  return 0;
}

// ---------------------------------------------------------------------------------------------
// the loss
// ---------------------------------------------------------------------------------------------
#define KDT_NT 512
// stats of a row, kept for the backward pass
// (maximum of the row, not yet times 1 / T, and sum; the teacher's log-sum-exp - without one: the largest kept logit - and mass; maximum
// and sum of what the sweep covered; M q_rest - p_rest, formed in 64 bits: where student and teacher agree it is a small difference
// of two numbers close to each other - without a rest: the sum of the kept logits' exponentials)
// Maxima are logits themselves, exact: the backward pass forms differences first, so logits far from zero lose nothing (a rounded
// logit / T of 1e6 would be 2^-5 off, 3 % of the probability).
enum { ST_TOP = 0, ST_SUM, ST_NORM, ST_MASS, ST_SWEEP_MAX, ST_SWEEP_SUM, ST_SHARE, ST_N };

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// NCH > 0: rows of up to NCH * 8 * KDT_NT elements are asked for before anything else and stay in registers.
// One read of the logits, bound by HBM and, nearly, by its vector instructions (as the selection): 5000 bf16 rows of 30 522 with 64 kept
// 76 us = 4.0 TB/s (median of 23, shortest 73), 12 000 155 us = 4.7 TB/s; 330 rows 11 us.
template <typename T, bool REST, int NCH>
__global__ __launch_bounds__(KDT_NT, sizeof(T) == 2 ? (REST ? 8 : 6) : 4) void kd_top_fwd_kernel(const T* __restrict__ s, int C, int64_t ld, const float* __restrict__ values,
                                                            const int32_t* __restrict__ classes, const float* __restrict__ lse_t,
                                                            int k, float inv_t, const float* __restrict__ roww,
                                                            float* __restrict__ stats, float* __restrict__ rowloss) {
  extern __shared__ uint32_t kept[];                         // REST: one bit per class
  __shared__ float red[16];
  __shared__ int cls[TOP_MAX_K];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  float* st = stats + r * ST_N;
  const float w = roww ? roww[r] : 1.0f;
  if (w == 0.f) {                                            // (block-uniform) a row of weight 0 takes no part, whatever it holds
    if (tid == 0) rowloss[r] = 0.f;
    return;
  }
  const T* x = s + r * ld;
  const int words = (C + 31) >> 5, chunks = (C + 7) >> 3;
  TopRaw8<T> keep[NCH > 0 ? NCH : 1];
  if constexpr (NCH > 0) {
#pragma unroll
    for (int n = 0; n < NCH; ++n)
      if (tid + n * KDT_NT < chunks) raw8<T>(x, tid + n * KDT_NT, C, -INFINITY, keep[n]);
  }
  // kept entries belong to the first wave: lane l holds entries l, l + 64, ..
  constexpr int NE = TOP_MAX_K / 64;
  int ci[NE];
  bool twice = false;                                        // this lane met a class that was marked already
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int j = tid + 64 * i;
      ci[i] = j < k ? classes[r * k + j] : -1;
      if (ci[i] < 0 || ci[i] >= C) ci[i] = -1;
    }
  }
  if constexpr (REST) {
    for (int i = tid; i < words; i += KDT_NT) kept[i] = 0u;
    __syncthreads();
    if (tid < 64) {
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        if (tid + 64 * i < k) cls[tid + 64 * i] = ci[i];
        const uint32_t bit = 1u << (ci[i] & 31);
        if (ci[i] >= 0) twice |= (atomicOr(&kept[ci[i] >> 5], bit) & bit) != 0;
      }
    }
    __syncthreads();
  }
  // maximum and sum of the row (REST: of the classes that are not kept), thread by thread
  auto drop_kept = [&](float (&v)[8], int c) __attribute__((always_inline)) {
    if constexpr (REST) {
      const uint32_t bits = (kept[c >> 2] >> (8 * (c & 3))) & 0xFFu;
      if (bits) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (bits >> e) & 1u ? -INFINITY : v[e];
      }
    }
  };
  float m = -INFINITY, sum = 0.f;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = tid + n * KDT_NT;
      if (c < chunks) {
        if constexpr (REST) {
          const uint32_t bits = (kept[c >> 2] >> (8 * (c & 3))) & 0xFFu;
          if (bits) keep[n].drop(bits);
        }
        m = fmaxf(m, max8(keep[n]));
      }
    }
  } else {
    for (int c = tid; c < chunks; c += KDT_NT) {
      float v[8];
      row8<T>(x, c, C, -INFINITY, v);
      drop_kept(v, c);
      m = fmaxf(m, max8(v));
    }
  }
  m = block_max(m, red);
  const ExpSum ex(m == -INFINITY ? 0.f : m, inv_t * TOP_LOG2E);
  auto sweep = [&](auto fast) __attribute__((always_inline)) {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int n = 0; n < NCH; ++n)
        if (tid + n * KDT_NT < chunks) {
          float v[8];
          keep[n].get(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += ex.template of<decltype(fast)::value>(v[e]);
        }
    } else {
      for (int c = tid; c < chunks; c += KDT_NT) {
        float v[8];
        row8<T>(x, c, C, -INFINITY, v);
        drop_kept(v, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += ex.template of<decltype(fast)::value>(v[e]);
      }
    }
  };
  if (ex.in_range) sweep(Yes()); else sweep(No());           // (block-uniform)
  float z[NE], y[NE];
  if (tid < 64) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      z[i] = ci[i] >= 0 ? values[r * k + tid + 64 * i] : 0.f;
      y[i] = ci[i] >= 0 ? to_f(x[ci[i]]) : 0.f;
    }
  }
  sum = block_sum(sum, red) * ex.tail();                     // (NaN where the row holds one)
  if (tid >= 64) return;                                     // the rest is the first wave's
  // A student close to its teacher has a loss of a few per thousand, the difference of terms of size 1, and p_rest is what is left
  // of 1: the k + 1 terms are formed in 64 bits (32 kept four digits of such a row's loss).
  // (Maximum, sum relative to it): a log-sum-exp in one number would lose the sum next to a maximum of the type's lowest value.
  const double t = (double)inv_t, m_sweep = (double)m * t;
  float raw_top = m;
  double top = m_sweep, total = (double)sum, swept = total;  // swept: the sum of what the sweep covered, relative to top
  double yd[NE], zd[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) { yd[i] = ci[i] >= 0 ? (double)y[i] * t : -INFINITY; zd[i] = ci[i] >= 0 ? (double)z[i] * t : -INFINITY; }
  if constexpr (REST) {                                      // + the kept classes, each once
    bool first[NE];
    double sk = 0.0;
    const bool dup = __any(twice);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      first[i] = ci[i] >= 0;
      if (64 * i < k && dup)
        for (int e = 0; e < k; ++e) first[i] = first[i] && !(e < tid + 64 * i && cls[e] == ci[i]);
      if (first[i]) raw_top = fmaxf(raw_top, y[i]);
    }
    raw_top = wave_max(raw_top);
    top = (double)raw_top * t;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64 * i < k && first[i] && top != -INFINITY) sk += exp(yd[i] - top);
    swept = m_sweep == -INFINITY ? (sum != sum ? (double)sum : 0.0) : (double)sum * exp(m_sweep - top);
    total = wave_sum_f64(sk) + swept;
  }
  const double ls = log(total);
  double norm, mass, p_rest = 0.0, p[NE] = {};
  float kept_norm, kept_sum = 0.f;                           // what the backward pass reads: see ST_NORM, ST_SHARE
  if constexpr (REST) {
    kept_norm = lse_t[r];
    norm = (double)kept_norm;
    mass = 0.0;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64 * i < k && zd[i] != -INFINITY) { p[i] = exp(zd[i] - norm); mass += p[i]; }
    mass = wave_sum_f64(mass);
    p_rest = mass != mass ? mass : (sum == 0.f ? 0.0 : fmax(0.0, 1.0 - mass));   // (sum == 0: no class is left for the rest)
  } else {
    double zs = 0.0;
    kept_norm = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (ci[i] >= 0) kept_norm = fmaxf(kept_norm, z[i]);
    kept_norm = wave_max(kept_norm);
    const double zm = (double)kept_norm * t;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64 * i < k && zd[i] != -INFINITY) { p[i] = exp(zd[i] - zm); zs += p[i]; }
    zs = wave_sum_f64(zs);
    kept_sum = (float)zs;
    norm = zm == -INFINITY ? -INFINITY : zm + log(zs);
    mass = zm == -INFINITY ? (zs != zs ? zs : 0.0) : (zs != zs ? zs : 1.0);
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64 * i < k && p[i] != 0.0) p[i] /= zs;
  }
  bool any = false;
#pragma unroll
  for (int i = 0; i < NE; ++i) any |= ci[i] >= 0;
  if (!__any(any)) { mass = p_rest = 0.0; }                  // a row without entries takes no part, whatever it holds
  double L = 0.0;
#pragma unroll
  for (int i = 0; i < NE; ++i)
    if (64 * i < k && p[i] != 0.0) L += p[i] * ((zd[i] - norm) - ((yd[i] - top) - ls));
  L = wave_sum_f64(L);
  if (tid == 0) {
    if (REST && p_rest != 0.0) L += p_rest * (log(p_rest) - ((m_sweep - top) + (log((double)sum) - ls)));
    rowloss[r] = w * (float)L;
    st[ST_TOP] = raw_top; st[ST_SUM] = (float)total; st[ST_NORM] = kept_norm; st[ST_MASS] = (float)(mass + p_rest);
    st[ST_SWEEP_MAX] = m; st[ST_SWEEP_SUM] = sum; st[ST_SHARE] = REST ? (float)((mass + p_rest) * (swept / total) - p_rest) : kept_sum;
  }
}
__global__ __launch_bounds__(1024) void kd_top_sum_kernel(const float* __restrict__ rowloss, int R, float coef, float* __restrict__ loss) {
  __shared__ float red[16];
  float s = 0.f;
  for (int r = threadIdx.x; r < R; r += 8192) {              // (8 loads on their way at a time)
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = rowloss[min(r + 1024 * u, R - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) s += r + 1024 * u < R ? v[u] : 0.f;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) loss[0] = s * coef;
}

template <typename T> __device__ __forceinline__ void store8_past(T* p, const float v[8]) {
  typedef T piece __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
  for (int h = 0; h < 8 / N; ++h) {
    piece t;
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = (T)v[N * h + e];
    __builtin_nontemporal_store(t, reinterpret_cast<piece*>(p) + h);
  }
}
// Gradient: one sweep writes every class as if none were kept, then the kept ones are written from their own formula (each
// duplicate of a class computes the same number).  The sweep's stores have arrived before the barrier between the two.
// Rows are taken from the last to the first: the forward sweep left the last ones in the 256 MB cache.  NT: a gradient that does not
// fit into that cache is stored past it, and the logits stay (bf16, 30 522 classes, 5000 rows, both directions: 198 us; with
// plain stores 207, first row first as well 213; 12 000 rows 453, 484, 488).  A smaller one is read from there by the next product.
// Bound by HBM: 118 us for 610 MB (5.2 TB/s; median of 23, the shortest 106).
template <typename T, bool REST, bool NT>
__global__ __launch_bounds__(KDT_NT) void kd_top_bwd_kernel(const T* __restrict__ s, int C, int64_t ld, const float* __restrict__ values,
                                                            const int32_t* __restrict__ classes, int k, float inv_t, float coef,
                                                            const float* __restrict__ roww, const float* __restrict__ stats,
                                                            const float* __restrict__ gout, T* __restrict__ ds, int64_t ldd, int acc) {
  __shared__ int cls[TOP_MAX_K];
  __shared__ float prob[TOP_MAX_K];
  const int tid = threadIdx.x;
  const int64_t r = gridDim.x - 1 - blockIdx.x;
  T* d = ds + r * ldd;
  const float w = roww ? roww[r] : 1.0f;
  const float* st = stats + r * ST_N;
  const int dchunks = (int)(ldd >> 3);                       // (ldd % 8 == 0, rows 16-byte aligned)
  if (w == 0.f || st[ST_MASS] == 0.f) {                      // (block-uniform) takes no part / no entries
    if (!acc) {
      const float zero[8] = {};
      for (int c = tid; c < dchunks; c += KDT_NT) store8<T>(d + 8 * (int64_t)c, zero);
    }
    return;
  }
  const float g = gout[0] * coef * w * inv_t;
  const float top = st[ST_TOP], total = st[ST_SUM], mass = st[ST_MASS], norm = st[ST_NORM];
  const T* x = s + r * ld;
  int ci = -1;
  float y = 0.f, before = 0.f;
  if (tid < k) {
    ci = classes[r * k + tid];
    if (ci < 0 || ci >= C) ci = -1;
    const float z = ci >= 0 ? values[r * k + tid] : -INFINITY;
    cls[tid] = ci;
    prob[tid] = z == -INFINITY ? 0.f : (REST ? expf(fmaf(z, inv_t, -norm)) : expf((z - norm) * inv_t) / st[ST_SHARE]);
    if (ci >= 0) {
      y = to_f(x[ci]);
      if (acc) before = to_f(d[ci]);
    }
  }
  __syncthreads();
  float mine = 0.f;
  if (ci >= 0) {
    float p = 0.f;
    for (int j = 0; j < k; ++j) p += cls[j] == ci ? prob[j] : 0.f;
    mine = g * (mass * (expf((y - top) * inv_t) / total) - p) + before;
  }
  // the others: f * exp((v - raw maximum) / T)
  const float c2 = inv_t * TOP_LOG2E, raw = st[ST_SWEEP_MAX], sweep = st[ST_SWEEP_SUM], base = raw == -INFINITY ? 0.f : raw;
  const float share = REST ? st[ST_SHARE] : mass;
  const float f = REST && sweep == 0.f ? 0.f : g * share / sweep;               // (no class is left: nothing is written that stays)
  for (int c = tid; c < dchunks; c += KDT_NT) {
    float v[8];
    row8<T>(x, c, C, -INFINITY, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 8 * c + e < C ? f * exp_diff(v[e], base, c2) : 0.f;
    if (acc) {
      float o[8];
      load8<T>(d + 8 * (int64_t)c, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += o[e];
    }
    if constexpr (NT) store8_past<T>(d + 8 * (int64_t)c, v);
    else store8<T>(d + 8 * (int64_t)c, v);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);                        // vmcnt(0)
  __syncthreads();
  if (ci >= 0) d[ci] = from_f<T>(mine);
}

static int kd_top_check(const char* name, int R, int C, int64_t ld, int k, float inv_t) {
  EVLM_REQUIRE(R > 0 && C > 0 && ld >= C, "%s: bad sizes", name);
  EVLM_REQUIRE(k > 0 && k <= TOP_MAX_K, "%s: k = %d is not in 1 .. %d", name, k, TOP_MAX_K);
  EVLM_REQUIRE(C <= (1 << 18), "%s: more than 2^18 classes", name);      // (one bit of LDS each: 32 KB)
  EVLM_REQUIRE(inv_t > 0.f && inv_t < 1e30f, "%s: the temperature must be positive and finite", name);
  return 0;
}
extern "C" int evlm_kl_top_fwd(int dtype, const void* s, int R, int C, int64_t ld, const float* values, const int32_t* classes,
                               const float* lse_t, int k, float inv_t, float weight, const float* row_weight, float* stats,
                               float* rowloss, float* loss, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = kd_top_check("evlm_kl_top_fwd", R, C, ld, k, inv_t)) return rc;
  EVLM_REQUIRE(s && values && classes && stats && rowloss && loss, "evlm_kl_top_fwd: null tensor");
  const size_t bits = (size_t)((C + 31) / 32) * 4;
#define KDT_FWD(REST, NCH, LDS) hipLaunchKernelGGL((kd_top_fwd_kernel<T, REST, NCH>), dim3(R), dim3(KDT_NT), LDS, stream, (const T*)s, C, ld, values, classes, lse_t, k, inv_t, row_weight, stats, rowloss)
  EVLM_DISPATCH_DTYPE(dtype, "evlm_kl_top_fwd",
    if (C <= 8 * 8 * KDT_NT) { if (lse_t) KDT_FWD(true, 8, bits); else KDT_FWD(false, 8, 0); }
    else { if (lse_t) KDT_FWD(true, 0, bits); else KDT_FWD(false, 0, 0); })
#undef KDT_FWD
  EVLM_LAUNCH_CHECK("evlm_kl_top_fwd");
  hipLaunchKernelGGL(kd_top_sum_kernel, dim3(1), dim3(1024), 0, stream, (const float*)rowloss, R, weight / (float)R, loss);
  EVLM_LAUNCH_CHECK("evlm_kl_top_fwd");
  return 0;
}
extern "C" int evlm_kl_top_bwd(int dtype, const void* s, int R, int C, int64_t ld, const float* values, const int32_t* classes,
                               int rest, int k, float inv_t, float weight, const float* row_weight, const float* stats,
                               const float* gout, void* ds, int64_t ldd, int accumulate, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = kd_top_check("evlm_kl_top_bwd", R, C, ld, k, inv_t)) return rc;
  EVLM_REQUIRE(s && values && classes && stats && gout && ds, "evlm_kl_top_bwd: null tensor");
  EVLM_REQUIRE(ldd >= C && ldd % 8 == 0 && ((uintptr_t)ds & 15) == 0, "evlm_kl_top_bwd: gradient rows must be whole aligned 16-byte pieces");
  const float coef = weight / (float)R;
#define KDT_BWD(REST, NT) hipLaunchKernelGGL((kd_top_bwd_kernel<T, REST, NT>), dim3(R), dim3(KDT_NT), 0, stream, (const T*)s, C, ld, values, classes, k, inv_t, coef, row_weight, stats, gout, (T*)ds, ldd, accumulate)
  EVLM_DISPATCH_DTYPE(dtype, "evlm_kl_top_bwd",
    const bool nt = !accumulate && (uint64_t)R * (uint64_t)ldd * sizeof(T) > ((uint64_t)256 << 20);
    if (rest) { if (nt) KDT_BWD(true, true); else KDT_BWD(true, false); }
    else { if (nt) KDT_BWD(false, true); else KDT_BWD(false, false); })
#undef KDT_BWD
  EVLM_LAUNCH_CHECK("evlm_kl_top_bwd");
  return 0;
}
